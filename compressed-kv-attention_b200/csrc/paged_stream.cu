// paged_stream.cu -- single-token attention over paged keys and values, up to 8 query rows at a
// time, and the combine pass that folds every row's partial states.
//
// A unit is up to 8 query rows and the tokens they share: the own pages of one sequence under one KV
// head or (batches of few rows) the shared prefix.  All units' 16-token tiles form one line, cut
// into equal runs, one for each warp of the grid, whatever the lengths are: a warp walks its run
// with an online softmax of its own and leaves one partial state per row for each unit it met.  No
// warp waits for another.
//
// The work is 4 bytes and 2 rows FMAs per K and V element, so it is bound by HBM; everything is
// arranged to keep loads in flight and nothing else in the way.  K and V go from global memory to
// the tensor cores' fragments without shared memory: the MMAs may take head dims (of QK) and output
// columns (of PV) in any order as long as both operands agree, so each lane loads 16 contiguous
// bytes of a token's row and calls them its fragment.
//   S = Q K^T (m16n8k16, rows 8-15 zero): lane (g, t) loads K token g, dims 32 j + 8 t .. + 7: words
//   0, 1 are the B fragment of k-step 2 j, words 2, 3 that of 2 j + 1; Q's A fragment is loaded the
//   same way.  The C fragment (query g, tokens 2 t, 2 t + 1) is already the B fragment of
//   O^T += V^T P^T, whose A fragment (dims x tokens) pairs two tokens' words by byte permutes:
//   lane (g, t) loads V tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 at dims 64 i + 8 g .. + 7.
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

// 16 (8) bytes that are read once.
__device__ __forceinline__ uint4 load16(const uint16_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load8(const uint16_t *p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + TT - 1) / TT; }

// A worker's stretch of one unit.
struct Unit {
    const int32_t *table;
    int64_t end;        // tile of the line after the unit's last
    int tokens;         // of the unit
    int skip;           // its tiles before the stretch
    int first, n;       // query rows first .. first + n - 1 of the head's (sequence, g) list
    int head;           // KV head
    int index;          // in the line
};

// The unit that tile f of the line belongs to.  starts[b]: tiles of one (head, group) of the
// sequences before b.
__device__ __forceinline__ Unit unit_at(const PagedArgs &a, const int32_t *starts, int64_t f) {
    Unit u;
    const int pt = tiles_of(a.prefix_len);
    const int64_t pre = int64_t(a.stream_prefix) * pt;
    if (f < pre) {
        u.index = int(f / pt);
        u.skip = int(f - int64_t(u.index) * pt);
        u.end = int64_t(u.index + 1) * pt;
        u.head = u.index / a.pre_groups;
        u.first = 8 * (u.index - u.head * a.pre_groups);
        u.n = min(8, a.batch * a.group - u.first);
        u.tokens = a.prefix_len;
        u.table = a.prefix_table;
        return u;
    }
    f -= pre;
    const int per = a.n_kv_heads * a.tail_groups;
    int lo = 0, hi = a.batch;  // starts[lo] * per <= f < starts[hi] * per
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (int64_t(starts[mid]) * per <= f) lo = mid;
        else hi = mid;
    }
    const int n = starts[lo + 1] - starts[lo];  // > 0: starts[lo + 1] * per > f
    const int64_t at = f - int64_t(starts[lo]) * per;
    const int k = int(at / n);
    u.skip = int(at - int64_t(k) * n);
    u.end = pre + int64_t(starts[lo]) * per + int64_t(k + 1) * n;
    u.head = k / a.tail_groups;
    const int qg = k - u.head * a.tail_groups;
    u.first = lo * a.group + 8 * qg;
    u.n = min(8, a.group - 8 * qg);
    u.tokens = tail_len(a, lo);
    u.table = a.table + int64_t(lo) * a.table_stride;
    u.index = a.stream_prefix + lo * per + k;
    return u;
}

// starts[b], b = 0 .. batch, from the lengths (every thread of the CTA).
__device__ __forceinline__ void scan_starts(const PagedArgs &a, int32_t *starts) {
    __shared__ int32_t part[NW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int32_t base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += NW * 32) {
        const int b = b0 + int(threadIdx.x);
        const int n = b < a.batch && a.max_len > 0 ? tiles_of(tail_len(a, b)) : 0;
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
        if (b < a.batch) starts[b] = before + s - n;
        base += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) starts[a.batch] = base;
    __syncthreads();
}

template <int D> struct Cfg {
    static constexpr int KJ = D / 32;                 // 32-dim pieces of a K row
    static constexpr int VI = D >= 64 ? D / 64 : 1;   // pieces of a V row
    static constexpr int VW = D >= 64 ? 4 : 2;        // words a lane loads of each
    static constexpr int NT = D <= 64 ? 128 / D : 1;  // tiles taken together: 8 KB in flight a warp
    static constexpr int CTAS = D <= 128 ? 2 : 1;
};

// BESIDE: launched behind the same call's prefix kernel, beside which it may run: that kernel's CTAs
// let it start once everything before them on the stream is complete, and it waits for them at its
// end, so that the combine pass, which waits for this grid, has both.
template <int D, int DT, bool BESIDE>
__global__ void __launch_bounds__(NW * 32, Cfg<D>::CTAS) stream_kernel(const PagedArgs a) {
    using C = Cfg<D>;
    constexpr int KJ = C::KJ, VI = C::VI, VW = C::VW, NT = C::NT;
    extern __shared__ int32_t starts[];
    if constexpr (!BESIDE) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    scan_starts(a, starts);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= a.batch; b += NW * 32) a.starts[b] = starts[b];
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int worker = int(blockIdx.x) * NW + int(threadIdx.x >> 5);
    const int64_t total = int64_t(a.stream_prefix) * tiles_of(a.prefix_len) +
                          int64_t(starts[a.batch]) * a.n_kv_heads * a.tail_groups;
    const int workers = stream_workers(a, total);
    int64_t f = worker < workers ? worker * total / workers : 0;
    const int64_t f_end = worker < workers ? (worker + 1) * total / workers : 0;
    while (f < f_end) {
        const Unit u = unit_at(a, starts, f);
        const int t0 = u.skip * TT;
        const int t1 = min(u.tokens, t0 + int(min(u.end, f_end) - f) * TT);
        f = u.end;

        // Q rows as A fragments
        uint4 qf[KJ];
        {
            const int r = u.first + (g < u.n ? g : 0), b = r / a.group;
            const uint16_t *q = a.q + int64_t(b) * a.q_token + int64_t(u.head * a.group + r - b * a.group) * a.q_head + 8 * t;
#pragma unroll
            for (int j = 0; j < KJ; ++j) qf[j] = load16(q + 32 * j);  // (rows past n repeat the first)
        }
        const uint16_t *kb = a.pool.k + int64_t(u.head) * a.pool.head_stride + 8 * t;
        const uint16_t *vb = a.pool.v + int64_t(u.head) * a.pool.head_stride + 2 * VW * g;
        float acc[VI * VW][4];
#pragma unroll
        for (int i = 0; i < VI * VW; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        float m = -INFINITY, l = 0.f;

        // The lanes look up the pages of the next tiles' tokens ahead of their use; nothing looks at an
        // entry before then, so its load is not waited for.  place -1: no such token.
        constexpr int LOOK = NT * TT > 32 ? 2 : 1;
        int32_t page[LOOK], place[LOOK];
        auto look_up = [&](int tok0) {
#pragma unroll
            for (int i = 0; i < LOOK; ++i) {
                const int tok = tok0 + 32 * i + (NT * TT >= 32 ? lane : lane & 15);
                page[i] = 0, place[i] = -1;
                if (tok < t1) {
                    int64_t at;
                    a.pool.split.at(tok, at, place[i]);
                    page[i] = __ldg(u.table + at);
                }
            }
        };
        look_up(t0);
        for (int tok = t0; tok < t1; tok += NT * TT) {
            // Rows of the tiles' tokens.  Where there is no token (the run's end, a bad entry) the pool's
            // first row is loaded in its place and then replaced by zeros: loads that depend on a
            // condition would be waited for one by one (3200 cycles an iteration).
            int64_t row[LOOK];
            uint32_t dead[LOOK];
#pragma unroll
            for (int i = 0; i < LOOK; ++i) {
                const bool in = place[i] >= 0, good = in && unsigned(page[i]) < unsigned(a.pool.n_pages);
                if (in && !good) report(a.status, KVX_ERR_RUNTIME, DERR_PAGE);
                row[i] = good ? int64_t(page[i]) * a.pool.page_stride + int64_t(place[i]) * a.pool.token_stride : 0;
                dead[i] = __ballot_sync(FULL, !good);  // (NT = 1: lanes 16-31 repeat lanes 0-15)
            }
            uint4 kf[NT][2][KJ];
            uint32_t vf[NT][4][VI][VW];
            auto load_k = [&]() {
#pragma unroll
                for (int k = 0; k < NT; ++k)
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const uint16_t *r = kb + __shfl_sync(FULL, row[k / 2], TT * (k & 1) + 8 * n + g);
#pragma unroll
                        for (int j = 0; j < KJ; ++j) kf[k][n][j] = load16(r + 32 * j);
                    }
            };
            auto load_v = [&]() {
#pragma unroll
                for (int k = 0; k < NT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t *r = vb + __shfl_sync(FULL, row[k / 2], TT * (k & 1) + 2 * t + (e & 1) + 8 * (e >> 1));
#pragma unroll
                        for (int i = 0; i < VI; ++i) {
                            if constexpr (VW == 4) {
                                const uint4 v = load16(r + 64 * i);
                                vf[k][e][i][0] = v.x, vf[k][e][i][1] = v.y, vf[k][e][i][2] = v.z, vf[k][e][i][3] = v.w;
                            } else {
                                const uint2 v = load8(r);
                                vf[k][e][i][0] = v.x, vf[k][e][i][1] = v.y;
                            }
                        }
                    }
            };
            load_k();
            if constexpr (D <= 128) load_v();  // (at 256 the registers hold one of K and V at a time)
            look_up(tok + NT * TT);

            float s[NT][2][4];
#pragma unroll
            for (int k = 0; k < NT; ++k)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    s[k][n][0] = s[k][n][1] = s[k][n][2] = s[k][n][3] = 0.f;
#pragma unroll
                    for (int j = 0; j < KJ; ++j) {
                        mma16<DT>(s[k][n], qf[j].x, 0u, qf[j].y, 0u, kf[k][n][j].x, kf[k][n][j].y);
                        mma16<DT>(s[k][n], qf[j].z, 0u, qf[j].w, 0u, kf[k][n][j].z, kf[k][n][j].w);
                    }
                }
            if constexpr (D > 128) load_v();
            // online softmax of query g: this lane has 4 of each tile's 16 tokens
#pragma unroll
            for (int k = 0; k < NT; ++k)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) s[k][n][e] *= a.scale_log2;
            if (LOOK == 2 ? (dead[0] | dead[LOOK - 1]) != 0u : dead[0] != 0u) {
#pragma unroll
                for (int k = 0; k < NT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int at = TT * (k & 1) + 2 * t + (e & 1) + 8 * (e >> 1);
                        if ((dead[k / 2] >> at) & 1u) {
                            s[k][e >> 1][e & 1] = -INFINITY;
#pragma unroll
                            for (int i = 0; i < VI; ++i)
#pragma unroll
                                for (int w = 0; w < VW; ++w) vf[k][e][i][w] = 0u;
                        }
                    }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < NT; ++k)
#pragma unroll
                for (int n = 0; n < 2; ++n) mx = fmaxf(mx, fmaxf(s[k][n][0], s[k][n][1]));
            if (__any_sync(FULL, mx > m)) {
                mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 2));
                const float mn = fmaxf(m, mx);
                const float al = mn == -INFINITY ? 1.f : exp2_sfu(m - mn);
                m = mn;
                l *= al;
                const float al0 = __shfl_sync(FULL, al, 8 * t), al1 = __shfl_sync(FULL, al, 8 * t + 4);
#pragma unroll
                for (int i = 0; i < VI * VW; ++i) acc[i][0] *= al0, acc[i][1] *= al1, acc[i][2] *= al0, acc[i][3] *= al1;
            }
            const float mu = m == -INFINITY ? 0.f : m - Elem<DT>::kBias;
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                uint32_t b[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float p0 = exp2_sfu(s[k][n][0] - mu), p1 = exp2_sfu(s[k][n][1] - mu);
                    l += p0 + p1;
                    b[n] = Elem<DT>::pack(p0, p1);
                }
#pragma unroll
                for (int i = 0; i < VI; ++i)
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        const uint32_t(&v)[4][VI][VW] = vf[k];
                        mma16<DT>(acc[i * VW + w], prmt(v[0][i][w], v[1][i][w], 0x5410u), prmt(v[0][i][w], v[1][i][w], 0x7632u),
                                  prmt(v[2][i][w], v[3][i][w], 0x5410u), prmt(v[2][i][w], v[3][i][w], 0x7632u), b[0], b[1]);
                    }
            }
        }

        // the part's state
        l += __shfl_xor_sync(FULL, l, 1);
        l += __shfl_xor_sync(FULL, l, 2);
        const int64_t out = a.stream_base + 8 * int64_t(worker + u.index);
        if (t == 0 && g < u.n) a.ml[out + g] = make_float2(m == -INFINITY ? m : m - Elem<DT>::kBias, l);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (2 * t + e >= u.n) continue;
            float *o = a.acc + (out + 2 * t + e) * D + 2 * VW * g;
#pragma unroll
            for (int i = 0; i < VI; ++i)
#pragma unroll
                for (int w = 0; w < VW; w += 2)
                    *reinterpret_cast<float4 *>(o + 64 * i + 2 * w) =
                        make_float4(acc[i * VW + w][e], acc[i * VW + w][2 + e], acc[i * VW + w + 1][e], acc[i * VW + w + 1][2 + e]);
        }
    }
    if constexpr (BESIDE) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Folds the partial states of one (sequence, head): M = max m_i, l = sum l_i 2^(m_i - M), out =
// (sum acc_i 2^(m_i - M)) / l.  One CTA per row; its warps take the parts in turn, each with a
// running maximum, so that no load waits for another's value; sums run in a fixed order.
constexpr int kCombineWarps = 8;
template <int D, int DT>
__global__ void __launch_bounds__(32 * kCombineWarps) combine_kernel(const PagedArgs a) {
    constexpr int V = D / 32;  // values per lane
    __shared__ float sacc[kCombineWarps][D];
    __shared__ float2 sml[kCombineWarps];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = blockIdx.y, h = blockIdx.x, head = h / a.group, gi = h - head * a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    // the row's parts: of the prefix (np, from row prow, pstep apart), then of its own tokens (ns)
    const int row = b * a.group + gi;
    int np = a.n_split, ns = 0;
    int64_t prow = int64_t(head) * a.n_split * a.row_pad + row, pstep = a.row_pad, srow = 0;
    if (a.stream_ctas > 0) {
        const int64_t pt = tiles_of(a.prefix_len), pre = a.stream_prefix * pt;
        const int per = a.n_kv_heads * a.tail_groups;
        const int64_t total = pre + int64_t(a.starts[a.batch]) * per;
        const int workers = stream_workers(a, total);
        // the workers that met tiles [f, f + n) of the line, and the first one's row of unit u;
        // worker_of(f) = the largest w with floor(w total / workers) <= f
        auto worker_of = [&](int64_t f) { return int(((f + 1) * workers - 1) / total); };
        auto parts = [&](int64_t f, int64_t n, int u, int64_t &first) {
            const int w = worker_of(f);
            first = a.stream_base + 8 * int64_t(w + u);
            return worker_of(f + n - 1) - w + 1;
        };
        if (a.stream_prefix > 0) {
            const int u = head * a.pre_groups + (row >> 3);
            np = parts(u * pt, pt, u, prow);
            prow += row & 7;
            pstep = 8;
        }
        const int n = a.starts[b + 1] - a.starts[b], k = head * a.tail_groups + (gi >> 3);
        if (n > 0) {
            ns = parts(pre + int64_t(a.starts[b]) * per + int64_t(k) * n, n, a.stream_prefix + b * per + k, srow);
            srow += gi & 7;
        }
    }
    float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll 4
    for (int i = warp; i < np + ns; i += nw) {
        const int64_t r = i < np ? prow + i * pstep : srow + 8 * int64_t(i - np);
        const float2 z = a.ml[r];
        const float *p = a.acc + r * D + V * lane;
        float v[V];
        if constexpr (V == 1) v[0] = p[0];
        else if constexpr (V == 2) {
            const float2 x = *reinterpret_cast<const float2 *>(p);
            v[0] = x.x, v[1] = x.y;
        } else {
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(p + j);
                v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
            }
        }
        const float mn = fmaxf(m, z.x);
        // (a part without a maximum has l = 0, or NaN, which stays)
        const float e = mn == -INFINITY ? 1.f : exp2_sfu(m - mn), w = z.x == -INFINITY ? 0.f : exp2_sfu(z.x - mn);
        m = mn;
        l = l * e + z.y * w;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = o[j] * e + (z.x == -INFINITY ? 0.f : w * v[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sacc[warp][V * lane + j] = o[j];
    if (lane == 0) sml[warp] = make_float2(m, l);
    __syncthreads();
    float M = -INFINITY;
    for (int w = 0; w < nw; ++w) M = fmaxf(M, sml[w].x);
    l = 0.f;
    float f[kCombineWarps];
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) {
        if (w >= nw) break;
        const float2 z = sml[w];
        f[w] = z.x == -INFINITY ? 0.f : exp2_sfu(z.x - M);
        l += z.y * f[w];
    }
    uint16_t *out = a.out + int64_t(b) * a.out_token + int64_t(h) * a.out_head;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kCombineWarps; ++w)
            if (w < nw) v += sacc[w][d] * f[w];
        out[d] = Elem<DT>::one(l == 0.f ? 0.f : v / l);
    }
    if (threadIdx.x == 0 && a.lse != nullptr)
        a.lse[int64_t(b) * a.n_q_heads + h] = l == 0.f ? -INFINITY : M * kPagedLn2 + logf(l);
}

template <int D, int DT, bool BESIDE> cudaError_t stream_launch(const PagedArgs &a, cudaStream_t s) {
    return launch_paged(stream_kernel<D, DT, BESIDE>, dim3(unsigned(a.stream_ctas)), NW * 32, 4 * (a.batch + 1), s, a);
}
template <int D, int DT> cudaError_t stream_d(const PagedArgs &a, cudaStream_t s) { return stream_launch<D, DT, false>(a, s); }
template <int D, int DT> cudaError_t beside_d(const PagedArgs &a, cudaStream_t s) { return stream_launch<D, DT, true>(a, s); }

template <int D, int DT> cudaError_t combine_d(const PagedArgs &a, cudaStream_t s) {
    // about this many parts a row: more warps where each would take several in turn
    const int units = a.stream_prefix + a.batch * a.n_kv_heads * a.tail_groups;
    const int parts = a.n_split + a.stream_ctas * NW / units;
    return launch_paged(combine_kernel<D, DT>, dim3(unsigned(a.n_q_heads), unsigned(a.batch)),
                        32 * (parts > 16 ? kCombineWarps : 4), 0, s, a);
}

}  // namespace

cudaError_t launch_paged_stream(int dim, int dtype, const PagedArgs &a, bool beside, cudaStream_t s) {
    if (a.stream_ctas <= 0) return cudaSuccess;
    if (beside) KVX_PAGED_DIM(beside_d)
    KVX_PAGED_DIM(stream_d)
}

cudaError_t launch_paged_combine(int dim, int dtype, const PagedArgs &a, cudaStream_t s) {
    if (a.batch <= 0) return cudaSuccess;
    KVX_PAGED_DIM(combine_d)
}

}  // namespace kvx
