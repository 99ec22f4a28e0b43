// paged_stream.cu -- single-token attention over paged keys and values, up to 8 query rows at a
// time, and the combine pass that folds every row's partial states.
//
// A unit is up to 8 query rows and the tokens they share: the own pages of one sequence under one KV
// head or (batches of few rows) the shared prefix.  A group of more than 8 query heads is several units,
// each of which reads the tokens: the first from HBM, the others from L2 as far as they are close enough behind it
// (64 sequences of up to 4096 tokens, 2 KV heads of 128: 33 us with 8 query heads each, 40 with 16).  All units' 16-token tiles form one line, with a
// margin after each for what a unit costs besides its tiles, cut into equal runs whatever the lengths
// are, one for each warp of the grid: a warp walks its run with an online softmax of its own and leaves
// one partial state per row for each unit it met.  No warp waits for another.  Where the kernel shares
// the device with the prefix kernel, the warps take runs from a counter instead, so that those that
// find room at once take more of them and the others what is left; which warp takes a run changes no
// result.
//
// The work is 4 bytes and 2 rows FMAs per K and V element, so it is bound by HBM (64 sequences of up to
// 4096 tokens, 8 KV heads of 128: 98 us with the combine pass, 5.5 TB/s; of up to 1024: 32 us, 4.2 TB/s,
// the ends of short runs); everything is arranged to keep loads in flight.  Each warp has a ring of stages of its own in shared memory (NT
// tiles of K and V rows, filled row by row with 16-byte asynchronous copies, the pages looked up one
// stage further ahead), so the copies of the next stages, the next unit's included, are in flight while
// one is computed.  (With the rows loaded into registers instead, a warp's tile took its load latency
// and its arithmetic in turn: 2.2 us on an idle device, and 16 warps a SM read 134 MB at 4.3 TB/s.)
// S^T = K Q^T (m16n8k16, tokens x queries) with K fragments by ldmatrix; its C fragment, packed and
// transposed by movmatrix, is the B fragment of O^T += V^T P^T, whose V^T fragments come by
// ldmatrix.trans.  Rows are 2 D + 16 bytes apart, so that eight of them meet no bank twice.
#include "paged_types.cuh"

namespace kvx {
namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int NW = kStreamWarps;
constexpr int TT = kStreamTile;

template <int DT>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
    if constexpr (DT == KVX_DTYPE_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + TT - 1) / TT; }

// Length of the line (less than 2^31, checked on the host) and of a run.
__device__ __forceinline__ int stream_line(const PagedArgs &a, int tail_line) {
    return a.stream_prefix * (tiles_of(a.prefix_len) + kUnitTiles) + tail_line * (a.n_kv_heads * a.tail_groups);
}
__device__ __forceinline__ int stream_run(const PagedArgs &a, int line) {
    return max(1, (line + a.stream_runs - 1) / a.stream_runs);
}

// A unit, and where it is on the line.
struct Unit {
    const int32_t *table;
    int at;             // position of its first tile
    int tokens;
    int first, n;       // query rows first .. first + n - 1 of the head's (sequence, g) list
    int head;           // KV head
    int index;          // among the units
    int b, k;           // sequence (-1: a prefix unit) and (head, group) in it
};

struct Line {
    const int32_t *starts, *lens;   // of the sequences (see scan_starts)
    int per, prefix, pre;           // units a sequence; positions of a prefix unit and of all of them
    __device__ __forceinline__ void of(const PagedArgs &a, const int32_t *starts_, const int32_t *lens_) {
        starts = starts_, lens = lens_;
        per = a.n_kv_heads * a.tail_groups;
        prefix = tiles_of(a.prefix_len) + kUnitTiles;
        pre = a.stream_prefix * prefix;
    }
    __device__ __forceinline__ Unit prefix_unit(const PagedArgs &a, int i) const {
        Unit u;
        u.index = i, u.at = i * prefix, u.b = -1, u.k = 0;
        u.head = i / a.pre_groups;
        u.first = 8 * (i - u.head * a.pre_groups);
        u.n = min(8, a.batch * a.group - u.first);
        u.tokens = a.prefix_len;
        u.table = a.prefix_table;
        return u;
    }
    __device__ __forceinline__ Unit tail_unit(const PagedArgs &a, int b, int k) const {
        Unit u;
        u.b = b, u.k = k, u.index = a.stream_prefix + b * per + k;
        u.tokens = lens[b];
        u.at = pre + starts[b] * per + k * (tiles_of(u.tokens) + kUnitTiles);
        u.head = a.tail_groups == 1 ? k : k / a.tail_groups;
        const int qg = k - u.head * a.tail_groups;
        u.first = b * a.group + 8 * qg;
        u.n = min(8, a.group - 8 * qg);
        u.table = a.table + int64_t(b) * a.table_stride;
        return u;
    }
    // The unit that position f is in.
    __device__ __forceinline__ Unit find(const PagedArgs &a, int f) const {
        if (f < pre) return prefix_unit(a, f / prefix);
        f -= pre;
        int lo = 0, hi = a.batch;  // starts[lo] * per <= f < starts[hi] * per
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] * per <= f) lo = mid;
            else hi = mid;
        }
        return tail_unit(a, lo, (f - starts[lo] * per) / (starts[lo + 1] - starts[lo]));
    }
    // The unit after u; false: there is none.
    __device__ __forceinline__ bool next(const PagedArgs &a, Unit &u) const {
        if (u.b < 0 && u.index + 1 < a.stream_prefix) {
            u = prefix_unit(a, u.index + 1);
            return true;
        }
        int b = u.b, k = u.k + 1;
        if (b < 0 || k == per) {
            k = 0;
            do {
                if (++b >= a.batch) return false;
            } while (lens[b] == 0);
        }
        u = tail_unit(a, b, k);
        return true;
    }
};

// The lengths, and starts[b], b = 0 .. batch: positions that one unit of every sequence before b takes
// (every thread of the CTA).
__device__ __forceinline__ void scan_starts(const PagedArgs &a, int32_t *starts, int32_t *lens) {
    __shared__ int32_t part[NW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int32_t base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += NW * 32) {
        const int b = b0 + int(threadIdx.x);
        const int len = b < a.batch && a.max_len > 0 ? tail_len(a, b) : 0, n = len > 0 ? tiles_of(len) + kUnitTiles : 0;
        int s = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(FULL, s, o);
            if (lane >= o) s += v;
        }
        if (lane == 31) part[warp] = s;
        __syncthreads();
        int before = base, all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += part[w];
            all += part[w];
        }
        if (b < a.batch) starts[b] = before + s - n, lens[b] = len;
        base += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) starts[a.batch] = base;
    __syncthreads();
}

template <int D> struct Cfg {
    static constexpr int KS = D / 16;                 // k-steps of QK, m-tiles of PV
    static constexpr int NT = D == 32 ? 2 : 1;        // tiles of a stage
    static constexpr int TOK = NT * TT;
    static constexpr int NS = D <= 64 ? 5 : 3;        // stages of a warp
    static constexpr int ROW = 2 * D + 16;            // bytes of a staged row
    static constexpr int O_V = TOK * ROW, O_DEAD = 2 * O_V;
    static constexpr int STAGE = O_DEAD + 16;
    static constexpr int RING = NS * STAGE;           // of a warp
    static constexpr int CTAS = D <= 128 ? 2 : 1;
    static_assert(TOK <= 32, "a lane for each token of a stage");
};

// A place in a run: its stages one after another.
struct Walk {
    Unit u;
    int tok, t1;    // the stage's first token, the end of the stretch
    int end;        // of the run
    bool more;
    // The stretch of u from position f on.
    __device__ __forceinline__ void stretch(int f) {
        tok = (f - u.at) * TT;
        t1 = min(u.tokens, (end - u.at) * TT);
    }
    __device__ __forceinline__ void begin(const PagedArgs &a, const Line &line, int f, int f_end) {
        end = f_end;
        u = line.find(a, f);
        more = true;
        stretch(f);
        if (tok >= u.tokens) next(a, line);  // the run begins in the unit's margin
    }
    __device__ __forceinline__ void next(const PagedArgs &a, const Line &line) {
        more = line.next(a, u) && u.at < end;
        if (more) stretch(u.at);
    }
};

// BESIDE: launched behind the same call's prefix kernel, beside which it may run: that kernel's CTAs
// let it start once everything before them on the stream is complete, and it waits for them at its
// end, so that the combine pass, which waits for this grid, has both.
template <int D, int DT, bool BESIDE>
__global__ void __launch_bounds__(NW * 32, Cfg<D>::CTAS) stream_kernel(const PagedArgs a) {
    using C = Cfg<D>;
    constexpr int KS = C::KS, NT = C::NT;
    extern __shared__ __align__(16) uint8_t smem[];
    int32_t *starts = reinterpret_cast<int32_t *>(smem + NW * C::RING), *lens = starts + a.batch + 1;
    if constexpr (!BESIDE) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // the warp's next run (in lane 0): fetched ahead, and not looked at before it is needed
    auto fetch = [&]() -> int { return !a.shared_runs ? INT_MAX : lane == 0 ? atomicAdd(a.next_run, 1) : 0; };
    int fetched = a.shared_runs ? fetch() : int(blockIdx.x) * NW + warp;
    scan_starts(a, starts, lens);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= a.batch; b += NW * 32) a.starts[b] = starts[b];
    // (the last unit's margin is no part of the line)
    const int total = max(0, stream_line(a, starts[a.batch]) - kUnitTiles), run = stream_run(a, total), runs = (total + run - 1) / run;
    Line line;
    line.of(a, starts, lens);
    const uint32_t ring = smem_u32(smem) + uint32_t(warp * C::RING);
    // the warp's next run that is not all margin, with a walk at its beginning; false: there is none
    auto take = [&](Walk &x, int &r) -> bool {
        for (;;) {
            r = __shfl_sync(FULL, fetched, 0);
            if (r >= runs) return false;
            fetched = fetch();
            x.begin(a, line, r * run, min(total, (r + 1) * run));
            if (x.more) return true;
        }
    };

    // ---- copies, NS - 1 stages ahead ----
    int r;
    Walk w, ahead;
    w.more = take(w, r);
    ahead = w;
    // runs that the copies have entered and the computation has not (a run has a stage at least; the
    // copies enter the next one as soon as they have issued a run's last)
    int queue[C::NS], queued = 0;
    auto cross = [&]() {
        int next;
        ahead.more = take(ahead, next);
        if (!ahead.more) return;
#pragma unroll
        for (int i = 0; i < C::NS; ++i)
            if (i == queued) queue[i] = next;
        ++queued;
    };
    // lane i: the page of token i from the lookup's first on (nothing looks at the entry before its stage is
    // issued, so its load is not waited for here) and its place in it (-1: no such token)
    int32_t page = 0, place = -1;
    auto look_up = [&]() {
        page = 0, place = -1;
        const int tok = ahead.tok + lane;
        if (ahead.more && tok < ahead.t1) {
            int64_t at;
            a.pool.split.at(tok, at, place);
            page = __ldg(ahead.u.table + at);
        }
    };
    look_up();
    int half = 0;  // which of the lookup's stages is next
    auto issue = [&](int stage) {
        if (ahead.more) {
            const bool in = place >= 0, good = in && unsigned(page) < unsigned(a.pool.n_pages);
            if (in && !good) report(a.status, KVX_ERR_RUNTIME, DERR_PAGE);
            const int64_t row = good ? int64_t(page) * a.pool.page_stride + int64_t(place) * a.pool.token_stride +
                                           int64_t(ahead.u.head) * a.pool.head_stride
                                     : -1;
            const uint32_t dead = __ballot_sync(FULL, !good) >> (half * C::TOK);
            const uint32_t dst = ring + uint32_t(stage % C::NS * C::STAGE);
            if (lane == 0) sts_u32(dst + C::O_DEAD, dead);
            constexpr int CH = D / 8, RPI = 32 / CH;  // pieces a row, rows a step
            const int c = lane % CH;
#pragma unroll
            for (int k = 0; k < C::TOK / RPI; ++k) {
                const int r = k * RPI + lane / CH;
                const int64_t o = __shfl_sync(FULL, row, half * C::TOK + r);
                const int64_t at = (o >= 0 ? o : 0) + 8 * c;
                copy16(dst + uint32_t(r * C::ROW + 16 * c), a.pool.k + at, o >= 0);
                copy16(dst + uint32_t(C::O_V + r * C::ROW + 16 * c), a.pool.v + at, o >= 0);
            }
            ahead.tok += C::TOK;
            ++half;
            if (ahead.tok >= ahead.t1) {
                ahead.next(a, line);
                if (!ahead.more) cross();
                half = 32;
            }
            if (half >= 32 / C::TOK) look_up(), half = 0;
        }
        copy_commit();
    };
#pragma unroll 1
    for (int i = 0; i < C::NS - 1; ++i) issue(i);

    // fragment addresses: lanes 8 i .. 8 i + 7 give the rows of matrix i
    const uint32_t k_at = uint32_t(((lane & 7) + ((lane >> 3) & 1) * 8) * C::ROW + (lane >> 4) * 16);
    const uint32_t v_at = uint32_t(C::O_V + ((lane & 7) + (lane >> 4) * 8) * C::ROW + ((lane >> 3) & 1) * 16);
    int stage = 0;
    while (w.more) {
        const Unit u = w.u;
        // Q rows as B fragments (rows past n repeat the first)
        uint32_t qf[KS][2];
        {
            const int r = u.first + (g < u.n ? g : 0), b = r / a.group;
            const uint16_t *q = a.q + int64_t(b) * a.q_token + int64_t(u.head * a.group + r - b * a.group) * a.q_head + 2 * t;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                qf[k][0] = __ldg(reinterpret_cast<const uint32_t *>(q + 16 * k));
                qf[k][1] = __ldg(reinterpret_cast<const uint32_t *>(q + 16 * k + 8));
            }
        }
        // lane (g, t): queries 2 t (m0, l0, acc[.][0, 2]) and 2 t + 1; acc[i]: dims 16 i + g, + 8
        float acc[KS][4];
#pragma unroll
        for (int i = 0; i < KS; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        for (; w.tok < w.t1; w.tok += C::TOK, ++stage) {
            __syncwarp();  // every lane has read the stage that is issued into next
            issue(stage + C::NS - 1);
            copy_wait<C::NS - 1>();
            __syncwarp();
            const uint32_t at = ring + uint32_t(stage % C::NS * C::STAGE);
            const uint32_t dead = lds_u32(at + C::O_DEAD);
            float s[NT][4];
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                float s2[2][4] = {};  // two chains
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t f[4];
                    ldsm_x4(at + k_at + uint32_t(k * TT * C::ROW + 32 * i), f[0], f[1], f[2], f[3]);
                    mma16<DT>(s2[i & 1], f[0], f[1], f[2], f[3], qf[i][0], qf[i][1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[k][e] = (s2[0][e] + s2[1][e]) * a.scale_log2;
            }
            if (dead != 0u) {  // (rows of zeros were stored)
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    if ((dead >> (TT * k + g)) & 1u) s[k][0] = s[k][1] = -INFINITY;
                    if ((dead >> (TT * k + g + 8)) & 1u) s[k][2] = s[k][3] = -INFINITY;
                }
            }
            float x0 = fmaxf(s[0][0], s[0][2]), x1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
            for (int k = 1; k < NT; ++k) x0 = fmaxf(x0, fmaxf(s[k][0], s[k][2])), x1 = fmaxf(x1, fmaxf(s[k][1], s[k][3]));
            if (__any_sync(FULL, x0 > m0 || x1 > m1)) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(FULL, x0, o));
                    x1 = fmaxf(x1, __shfl_xor_sync(FULL, x1, o));
                }
                x0 = fmaxf(x0, m0), x1 = fmaxf(x1, m1);
                const float e0 = x0 == -INFINITY ? 1.f : exp2_sfu(m0 - x0), e1 = x1 == -INFINITY ? 1.f : exp2_sfu(m1 - x1);
                m0 = x0, m1 = x1;
                l0 *= e0, l1 *= e1;
#pragma unroll
                for (int i = 0; i < KS; ++i) acc[i][0] *= e0, acc[i][1] *= e1, acc[i][2] *= e0, acc[i][3] *= e1;
            }
            const float u0 = m0 == -INFINITY ? 0.f : m0 - Elem<DT>::kBias, u1 = m1 == -INFINITY ? 0.f : m1 - Elem<DT>::kBias;
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                const float p0 = exp2_sfu(s[k][0] - u0), p1 = exp2_sfu(s[k][1] - u1), p2 = exp2_sfu(s[k][2] - u0),
                            p3 = exp2_sfu(s[k][3] - u1);
                l0 += p0 + p2, l1 += p1 + p3;
                const uint32_t b0 = movm_t(Elem<DT>::pack(p0, p1)), b1 = movm_t(Elem<DT>::pack(p2, p3));
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t f[4];
                    ldsm_x4_t(at + v_at + uint32_t(k * TT * C::ROW + 32 * i), f[0], f[1], f[2], f[3]);
                    mma16<DT>(acc[i], f[0], f[1], f[2], f[3], b0, b1);
                }
            }
        }

        // the part's state
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            l0 += __shfl_xor_sync(FULL, l0, o);
            l1 += __shfl_xor_sync(FULL, l1, o);
        }
        const int64_t out = a.stream_base + 8 * int64_t(r + u.index);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (2 * t + e >= u.n) continue;
            const float m = e ? m1 : m0;
            if (g == 0) a.ml[out + 2 * t + e] = make_float2(m == -INFINITY ? m : m - Elem<DT>::kBias, e ? l1 : l0);
            float *o = a.acc + (out + 2 * t + e) * D + g;
#pragma unroll
            for (int i = 0; i < KS; ++i) o[16 * i] = acc[i][e], o[16 * i + 8] = acc[i][2 + e];
        }
        w.next(a, line);
        if (!w.more && queued > 0) {
            r = queue[0];
#pragma unroll
            for (int i = 0; i + 1 < C::NS; ++i) queue[i] = queue[i + 1];
            --queued;
            w.begin(a, line, r * run, min(total, (r + 1) * run));
        }
    }
    copy_wait<0>();
    if constexpr (BESIDE) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Folds the partial states of one (sequence, head): M = max m_i, l = sum l_i 2^(m_i - M), out =
// (sum acc_i 2^(m_i - M)) / l.  One CTA per row; its warps take the parts in turn, a few parts' loads at
// a time and each with a running maximum, so that no load waits for another's value; sums run in a
// fixed order.  2048 rows of 18 parts of 128 values (19 MB from L2) take 6.5 us, 28 rows of 64
// values 4.1, most of it the launch.
template <int V> struct Fold {
    static constexpr int U = V <= 4 ? 4 : 2;  // parts loaded together
    float m = -INFINITY, l = 0.f, o[V] = {};
    // Parts i, i + step, ... of `n` in rows first, first + stride, ...
    template <int D>
    __device__ __forceinline__ void take(const PagedArgs &a, int64_t first, int64_t stride, int n, int i, int step, int lane) {
        for (; i < n; i += U * step) {
            float2 z[U];
            float v[U][V];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int64_t r = first + int64_t(min(i + k * step, n - 1)) * stride;
                z[k] = a.ml[r];
                const float *p = a.acc + r * D + V * lane;
                if constexpr (V == 1) v[k][0] = p[0];
                else if constexpr (V == 2) {
                    const float2 x = *reinterpret_cast<const float2 *>(p);
                    v[k][0] = x.x, v[k][1] = x.y;
                } else {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const float4 x = *reinterpret_cast<const float4 *>(p + j);
                        v[k][j] = x.x, v[k][j + 1] = x.y, v[k][j + 2] = x.z, v[k][j + 3] = x.w;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (i + k * step < n) {
                    const float mn = fmaxf(m, z[k].x);
                    // (a part without a maximum has l = 0, or NaN, which stays)
                    const float e = mn == -INFINITY ? 1.f : exp2_sfu(m - mn), w = z[k].x == -INFINITY ? 0.f : exp2_sfu(z[k].x - mn);
                    m = mn;
                    l = l * e + z[k].y * w;
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] = o[j] * e + (z[k].x == -INFINITY ? 0.f : w * v[k][j]);
                }
        }
    }
};

constexpr int kCombineWarps = 8;
template <int D, int DT>
__global__ void __launch_bounds__(32 * kCombineWarps) combine_kernel(const PagedArgs a) {
    constexpr int V = D / 32;  // values per lane
    __shared__ float sacc[kCombineWarps][D];
    __shared__ float2 sml[kCombineWarps];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (a.shared_runs && blockIdx.x + blockIdx.y + threadIdx.x == 0) *a.next_run = 0;  // for the next call
    const int b = blockIdx.y, h = blockIdx.x, head = h / a.group, gi = h - head * a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int row = b * a.group + gi;
    // (the line's lengths, for the streamed parts, are on their way while the prefix's parts are folded)
    int s0 = 0, s1 = 0, s_end = 0;
    if (a.stream_ctas > 0) s0 = a.starts[b], s1 = a.starts[b + 1], s_end = a.starts[a.batch];
    Fold<V> f;
    if (a.n_split > 0) f.template take<D>(a, int64_t(head) * a.n_split * a.row_pad + row, a.row_pad, a.n_split, warp, nw, lane);
    if (a.stream_ctas > 0) {
        const int n = s1 - s0 - kUnitTiles;  // the sequence's tiles (< 0: none)
        const int run = stream_run(a, max(0, stream_line(a, s_end) - kUnitTiles));
        const int pt = tiles_of(a.prefix_len), per = a.n_kv_heads * a.tail_groups;
        // the runs that met tiles [at, at + n) of the line left rows of unit u from the first one's on
        auto fold_unit = [&](int at, int n, int u, int g) {
            const int w = at / run;
            f.template take<D>(a, a.stream_base + 8 * (int64_t(w) + u) + g, 8, (at + n - 1) / run - w + 1, warp, nw, lane);
        };
        if (a.stream_prefix > 0) {
            const int u = head * a.pre_groups + (row >> 3);
            fold_unit(u * (pt + kUnitTiles), pt, u, row & 7);
        }
        const int k = head * a.tail_groups + (gi >> 3);
        if (n > 0)
            fold_unit(a.stream_prefix * (pt + kUnitTiles) + s0 * per + k * (n + kUnitTiles), n, a.stream_prefix + b * per + k, gi & 7);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sacc[warp][V * lane + j] = f.o[j];
    if (lane == 0) sml[warp] = make_float2(f.m, f.l);
    __syncthreads();
    float M = -INFINITY, l = 0.f, w8[kCombineWarps];
    for (int w = 0; w < nw; ++w) M = fmaxf(M, sml[w].x);
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) {
        w8[w] = 0.f;
        if (w >= nw) continue;
        const float2 z = sml[w];
        if (z.x != -INFINITY) w8[w] = exp2_sfu(z.x - M);
        l += z.y * w8[w];
    }
    uint16_t *out = a.out + int64_t(b) * a.out_token + int64_t(h) * a.out_head;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kCombineWarps; ++w)
            if (w < nw) v += sacc[w][d] * w8[w];
        out[d] = Elem<DT>::one(l == 0.f ? 0.f : v / l);
    }
    if (threadIdx.x == 0 && a.lse != nullptr)
        a.lse[int64_t(b) * a.n_q_heads + h] = l == 0.f ? -INFINITY : M * kPagedLn2 + logf(l);
}

constexpr int list_bytes(int batch) { return 8 * batch + 4; }   // of scan_starts
template <int D, int DT> cudaError_t prepare_d() {
    const int bytes = NW * Cfg<D>::RING + list_bytes(kMaxStreamBatch);
    const cudaError_t e = allow_smem(stream_kernel<D, DT, false>, bytes);
    return e != cudaSuccess ? e : allow_smem(stream_kernel<D, DT, true>, bytes);
}
template <int D, int DT, bool BESIDE> cudaError_t stream_launch(const PagedArgs &a, cudaStream_t s) {
    return launch_paged(stream_kernel<D, DT, BESIDE>, dim3(unsigned(a.stream_ctas)), NW * 32, NW * Cfg<D>::RING + list_bytes(a.batch), s, a);
}
template <int D, int DT> cudaError_t stream_d(const PagedArgs &a, cudaStream_t s) { return stream_launch<D, DT, false>(a, s); }
template <int D, int DT> cudaError_t beside_d(const PagedArgs &a, cudaStream_t s) { return stream_launch<D, DT, true>(a, s); }

template <int D, int DT> cudaError_t combine_d(const PagedArgs &a, cudaStream_t s) {
    // about this many parts a row: as many warps as take them in two rounds of loads (a fold of 14 heads
    // by 16 rows of 3 parts: 2 warps 5.0 us, 4 warps 5.8; of 32 by 5 of 22 at dim 256: 8 warps 5.7, 4 warps 7.1)
    const int units = a.stream_prefix + a.batch * a.n_kv_heads * a.tail_groups;
    const int parts = a.n_split + a.stream_runs / units;
    return launch_paged(combine_kernel<D, DT>, dim3(unsigned(a.n_q_heads), unsigned(a.batch)),
                        32 * (parts > 8 * Fold<D / 32>::U ? kCombineWarps : parts > 8 ? 4 : 2), 0, s, a);
}

}  // namespace

cudaError_t prepare_paged_stream(int dim, int dtype) { KVX_PAGED_DIM(prepare_d) }

cudaError_t launch_paged_stream(int dim, int dtype, const PagedArgs &a, bool beside, cudaStream_t s) {
    if (a.stream_ctas <= 0) return cudaSuccess;
    if (beside) KVX_PAGED_DIM(beside_d, a, s)
    KVX_PAGED_DIM(stream_d, a, s)
}

cudaError_t launch_paged_combine(int dim, int dtype, const PagedArgs &a, cudaStream_t s) {
    if (a.batch <= 0) return cudaSuccess;
    KVX_PAGED_DIM(combine_d, a, s)
}

}  // namespace kvx
