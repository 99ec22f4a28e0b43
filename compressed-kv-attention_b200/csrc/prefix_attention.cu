// prefix_attention.cu -- attention of many query rows over one shared prefix, on the fifth-generation
// tensor cores.
//
// Every (sequence, query head) of a KV head is a row of one matrix: S = Q K^T and O += P V with up
// to 128 rows a CTA, so a piece of the prefix is read once for 128 rows.  One CTA takes one item:
// a KV head, 128 of its rows and a run of 64-token tiles; it leaves one partial state per row.
//
//  * Warps 4-6 load: each K or V tile goes by 16-byte asynchronous copies into a slot of a
//    shared-memory ring in the layout the tensor cores read (rows of 128 bytes, 16-byte pieces
//    XOR-swizzled by the row; 64-byte rows at D = 32).  Copies by row take pages of any length and
//    strides, and fill the rows past the run's end with zeros.
//  * Warp 7 issues the MMAs (one thread): S(i) = Q K(i)^T into one of two TMEM buffers, then
//    O += P(i - 1) V(i - 1) with P read from TMEM (it replaces S there), so that S(i) is computed
//    while the softmax of tile i - 1 runs.  V is the N-major operand: the same rows as stored.
//  * Warps 0-3 do the softmax, a thread to a row: no shuffles.  The maximum that weights are
//    relative to is raised, and O rescaled in TMEM, only when some row's scores pass it by 2^8
//    (2^5 for FP16 weights), which is rare after the first tile; l and O share it, so it cancels.
//
// What bounds it: per 64-token tile and 128 rows the SM's exponentials take 64 x 128 / 16 = 512
// cycles, the MMAs 4 D (256 at D = 64, 512 at D = 128) and the tile's bytes from HBM 256 D / 23
// (712 at D = 64, 1425 at D = 128, shared by all 128-row items of the head through L2).  Two CTAs
// a SM (one at D = 256) overlap one's softmax with the other's waits.
#include "paged_types.cuh"

namespace kvx {
namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int TT = kPrefixTile;         // tokens per tile
constexpr int ROWS = kPrefixRows;       // query rows per item
constexpr int SW = 4, LW = 3;           // softmax and loader warps
constexpr int THREADS = 32 * (SW + LW + 1);
constexpr uint32_t kWaitUs = 1000000;   // bounded waits

template <int D> struct Cfg {
    static constexpr int ROWB = D >= 64 ? 128 : 64;         // bytes of a row of one panel of head dims
    static constexpr int SLOT = TT * D * 2;
    static constexpr int NSLOT = D == 32 ? 12 : (D == 64 ? 10 : 5);
    static constexpr int LAG = NSLOT - 2;                   // tiles in flight before one is announced
    static constexpr int CTAS = D == 256 ? 1 : 2;           // per SM
    static constexpr int O_Q = 0;
    static constexpr int O_RING = ROWS * D * 2;
    static constexpr int O_BAR = O_RING + NSLOT * SLOT;
    static constexpr int SMEM = O_BAR + 16 * NSLOT + 64;
    static constexpr int LDO = D + 4;                       // floats of a staged output row
    static constexpr int TMEM = D == 256 ? 512 : 256;       // columns: O at 0, S / P buffers at D, D + 64
    static constexpr uint64_t LAYOUT = D >= 64 ? 2 : 4;     // 128- / 64-byte swizzle
    static_assert(ROWS * LDO * 4 <= O_BAR, "the staged outputs fit where Q and the ring were");
    static_assert(D + 2 * TT <= TMEM && CTAS * TMEM <= 512, "TMEM columns");
    static_assert(CTAS * (SMEM + 1024) <= 233472, "shared memory");
};

// Byte of 16-byte piece c of row r in a tile of R rows.
template <int D, int R> __device__ __forceinline__ uint32_t tile_off(int r, int c) {
    if constexpr (D >= 64) return uint32_t((c >> 3) * (R * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    else return uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// Shared-memory matrix descriptor: start address, leading and stride byte offsets (all / 16),
// descriptor version 1 (sm_100), swizzle mode.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride, uint64_t layout) {
    return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(lead >> 4) << 16) | (uint64_t(stride >> 4) << 32) |
           (uint64_t(1) << 46) | (layout << 61);
}

// Instruction descriptor: FP32 accumulator, A and B of the cache's type, A K-major, B K-major or
// N-major, N columns, 128 rows.
template <int DT> __device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool b_n_major) {
    const uint32_t t = DT == KVX_DTYPE_BF16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (b_n_major ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) |
           (uint32_t(ROWS >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// Arrive on `bar` when every MMA issued so far by this thread has completed.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Waits for the loads and names their registers, so that no use of them moves above it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 16 bytes global -> shared, zeros when there is no such row.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Barriers of a CTA (8 bytes each): full and empty of every ring slot, then these.
enum { B_S0, B_S1, B_P0, B_P1, B_PV, B_Q, B_COUNT };

// One item.
struct Item {
    int head, first, n;   // KV head, first row, rows
    int t0, t1, tiles;
    int64_t row0;
};
__device__ __forceinline__ Item item_of(const PagedArgs &a, int i) {
    Item x;
    const int mt = i % a.row_groups;  // 128-row groups of one piece of the prefix run together
    i /= a.row_groups;
    const int s = i % a.n_split;
    x.head = i / a.n_split;
    x.first = mt * ROWS;
    x.n = min(ROWS, a.batch * a.group - x.first);
    x.t0 = s * a.split_tokens;
    x.t1 = min(a.prefix_len, x.t0 + a.split_tokens);
    x.tiles = (x.t1 - x.t0 + TT - 1) / TT;
    x.row0 = int64_t(x.head * a.n_split + s) * a.row_pad + x.first;
    return x;
}

// The ring's order: K0, K1, V0, K2, V1, ..., K(n-1), V(n-2), V(n-1).
__device__ __forceinline__ int k_item(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int v_item(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }

template <int D, int DT>
__global__ void __launch_bounds__(THREADS, Cfg<D>::CTAS) prefix_kernel(const PagedArgs a) {
    using C = Cfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    volatile uint32_t *tmem_base = reinterpret_cast<volatile uint32_t *>(smem + C::O_BAR + 16 * C::NSLOT + 8 * B_COUNT);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sb = smem_u32(smem);
    const uint32_t bars = sb + C::O_BAR;
    auto full = [&](int q) { return bars + 8u * uint32_t(q % C::NSLOT); };
    auto empty = [&](int q) { return bars + 8u * uint32_t(C::NSLOT + q % C::NSLOT); };
    auto bar = [&](int b) { return bars + 8u * uint32_t(2 * C::NSLOT + b); };
    const Item it = item_of(a, int(blockIdx.x));
    auto wait = [&](uint32_t b, int phase) -> bool {
        if (mbar_wait_bounded(b, uint32_t(phase & 1), kWaitUs)) return true;
        report(a.status, KVX_ERR_TIMEOUT, DERR_TIMEOUT);
        return false;
    };

    if (warp == SW + LW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar(B_COUNT)),
                     "n"(C::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NSLOT; ++i) mbar_init(full(i), LW), mbar_init(empty(i), 1);
        mbar_init(bar(B_S0), 1), mbar_init(bar(B_S1), 1), mbar_init(bar(B_P0), SW), mbar_init(bar(B_P1), SW);
        mbar_init(bar(B_PV), 1), mbar_init(bar(B_Q), SW);
        fence_mbar_init();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base;

    if (warp >= SW && warp < SW + LW) {
        // ---- loads ----
        // Loader warp w copies rows w, w + LW, ... of every tile: lane k holds the offset of row w +
        // LW k (-1: no such token), looked up a tile ahead of its use.
        constexpr int CH = D / 8, RPS = 32 / CH;              // pieces a row, rows a step
        constexpr int MINE = (TT + LW - 1) / LW, STEPS = (MINE + RPS - 1) / RPS;
        const int w = warp - SW, c = lane % CH;
        const int64_t head = int64_t(it.head) * a.pool.head_stride + 8 * c;
        auto look_up = [&](int tile) -> int64_t {
            const int r = w + LW * lane, tok = it.t0 + tile * TT + r;
            return r < TT && tok < it.t1 ? page_row(a.pool, a.prefix_table, tok, a.status) : -1;
        };
        auto announce = [&](int i) {
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(full(i));
        };
        // rows of the latest K tile, of the one before it (V follows a tile behind) and of the next
        int64_t r_k = -1, r_before = -1, r_next = look_up(0);
        bool ok = true;
        int q = 0;
        for (; q < 2 * it.tiles; ++q) {
            const bool last = q == 2 * it.tiles - 1, is_v = last || (q > 0 && (q & 1) == 0);
            if (!is_v) {
                r_before = r_k;
                r_k = r_next;
                r_next = look_up((q + 1) / 2 + 1);
            }
            if (q >= C::NSLOT) ok = __all_sync(FULL, wait(empty(q), q / C::NSLOT - 1));
            if (!ok) break;
            const uint16_t *src = (is_v ? a.pool.v : a.pool.k) + head;
            const uint32_t dst = sb + uint32_t(C::O_RING + (q % C::NSLOT) * C::SLOT);
            const int64_t mine = is_v && !last ? r_before : r_k;
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                const int k = j * RPS + lane / CH, r = w + LW * k;
                const int64_t o = __shfl_sync(FULL, mine, k);
                if (r < TT) copy16(dst + tile_off<D, TT>(r, c), src + (o >= 0 ? o : 0), o >= 0);
            }
            copy_commit();
            if (q >= C::LAG) {
                copy_wait<C::LAG>();
                announce(q - C::LAG);
            }
        }
        copy_wait<0>();
        if (ok)
            for (int i = max(0, q - C::LAG); i < q; ++i) announce(i);
    } else if (warp == SW + LW) {
        // ---- MMAs ----
        if (lane == 0 && wait(bar(B_Q), 0)) {
            constexpr uint32_t qk = instr_desc<DT>(TT, false), pv = instr_desc<DT>(D, true);
            constexpr uint32_t K8 = 8 * C::ROWB;  // bytes of 8 rows
            for (int i = 0; i <= it.tiles; ++i) {
                if (i < it.tiles) {
                    const int x = k_item(i);
                    if (!wait(full(x), x / C::NSLOT)) break;
                    fence_after();
                    const uint32_t kq = sb + C::O_Q, kk = sb + uint32_t(C::O_RING + (x % C::NSLOT) * C::SLOT);
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        const uint32_t p = uint32_t(s / (C::ROWB / 32)), o = uint32_t(s % (C::ROWB / 32)) * 32;
                        mma_ss(tm + D + (i & 1) * TT, smem_desc(kq + p * (ROWS * C::ROWB) + o, 16, K8, C::LAYOUT),
                               smem_desc(kk + p * (TT * C::ROWB) + o, 16, K8, C::LAYOUT), qk, s > 0);
                    }
                    mma_commit(empty(x));
                    mma_commit(bar(B_S0 + (i & 1)));
                }
                if (i > 0) {
                    const int j = i - 1, x = v_item(j, it.tiles);
                    if (!wait(full(x), x / C::NSLOT) || !wait(bar(B_P0 + (j & 1)), j >> 1)) break;
                    fence_after();
                    const uint32_t vv = sb + uint32_t(C::O_RING + (x % C::NSLOT) * C::SLOT);
#pragma unroll
                    for (int s = 0; s < TT / 16; ++s)
                        mma_ts(tm, tm + D + (j & 1) * TT + 8 * s, smem_desc(vv + 2 * s * K8, TT * C::ROWB, K8, C::LAYOUT),
                               pv, j > 0 || s > 0);
                    mma_commit(empty(x));
                    mma_commit(bar(B_PV));
                }
            }
        }
        __syncwarp();
    } else {
        // ---- Q, then the softmax ----
        constexpr int CH = D / 8;
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * CH; i += 32 * SW) {
            const int r = i / CH, c = i % CH;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (r < it.n) {
                const int row = it.first + r, b = row / a.group, h = it.head * a.group + row - b * a.group;
                v = *reinterpret_cast<const uint4 *>(a.q + int64_t(b) * a.q_token + int64_t(h) * a.q_head + 8 * c);
            }
            sts_v4(sb + C::O_Q + tile_off<D, ROWS>(r, c), v.x, v.y, v.z, v.w);
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_Q));

        const bool live = 32 * warp < it.n;  // rows past the item's are not computed
        const uint32_t lanes = uint32_t(warp * 32) << 16;
        constexpr float kGrow = DT == KVX_DTYPE_BF16 ? 8.f : 15.f - Elem<DT>::kBias;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int i = 0; i < it.tiles && ok; ++i) {
            ok = __all_sync(FULL, wait(bar(B_S0 + (i & 1)), i >> 1));
            if (!ok) break;
            fence_after();
            bool pv_seen = i == 0;  // PV(i - 1) has completed
            if (live) {
                const uint32_t st = tm + lanes + uint32_t(D + (i & 1) * TT);
                uint32_t x0[32], x1[32];
                tmem_ld32(st, x0);
                tmem_ld32(st + 32, x1);
                tmem_wait_ld(x0);
                tmem_wait_ld(x1);
                const int valid = it.t1 - (it.t0 + i * TT);
                if (valid < TT) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if (j >= valid) x0[j] = 0xFF800000u;
                        if (j + 32 >= valid) x1[j] = 0xFF800000u;
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < 32; ++j) mx = fmaxf(mx, fmaxf(__uint_as_float(x0[j]), __uint_as_float(x1[j])));
                mx *= a.scale_log2;
                if (__any_sync(FULL, mx > m + kGrow || (m == -INFINITY && mx > m))) {
                    const float mn = fmaxf(m, mx);
                    const float al = mn == -INFINITY ? 1.f : exp2_sfu(m - mn);
                    m = mn;
                    l *= al;
                    if (i > 0) {
                        // O is complete up to tile i - 1, and the next PV waits for this warp
                        ok = __all_sync(FULL, wait(bar(B_PV), i - 1));
                        if (!ok) break;
                        pv_seen = true;
                        fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(tm + lanes + c, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * al);
                            tmem_st32(tm + lanes + c, o);
                        }
                    }
                }
                const float mu = m == -INFINITY ? 0.f : m - Elem<DT>::kBias;
                uint32_t p[32];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float u = exp2_sfu(__fmaf_rn(__uint_as_float(x0[2 * j]), a.scale_log2, -mu));
                    const float v = exp2_sfu(__fmaf_rn(__uint_as_float(x0[2 * j + 1]), a.scale_log2, -mu));
                    const float w = exp2_sfu(__fmaf_rn(__uint_as_float(x1[2 * j]), a.scale_log2, -mu));
                    const float z = exp2_sfu(__fmaf_rn(__uint_as_float(x1[2 * j + 1]), a.scale_log2, -mu));
                    p[j] = Elem<DT>::pack(u, v);
                    p[16 + j] = Elem<DT>::pack(w, z);
                    l += (u + v) + (w + z);
                }
                tmem_st32(st, p);
                tmem_wait_st();
            }
            // B_PV is waited for once a tile, before the arrival that lets its next phase begin: a
            // phase later its parity would not tell PV(i - 1) done from PV(i) to come
            if (!pv_seen) ok = __all_sync(FULL, wait(bar(B_PV), i - 1));
            if (!ok) break;
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_P0 + (i & 1)));
        }
        if (ok) ok = __all_sync(FULL, wait(bar(B_PV), it.tiles - 1));
        if (ok && live) {
            // every copy and MMA of the CTA has completed: Q and the ring make room for the rows
            fence_after();
            float *stage = reinterpret_cast<float *>(smem) + warp * 32 * C::LDO;
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(tm + lanes + c, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                    *reinterpret_cast<uint4 *>(stage + lane * C::LDO + c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            }
            __syncwarp();
            const int n = min(32, it.n - 32 * warp);
            float *dst = a.acc + (it.row0 + 32 * warp) * D;
            for (int j = lane; j < n * (D / 4); j += 32)
                reinterpret_cast<float4 *>(dst)[j] =
                    *reinterpret_cast<const float4 *>(stage + (j / (D / 4)) * C::LDO + 4 * (j % (D / 4)));
            if (lane < n) a.ml[it.row0 + 32 * warp + lane] = make_float2(m == -INFINITY ? m : m - Elem<DT>::kBias, l);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == SW + LW)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(C::TMEM) : "memory");
}

template <int D, int DT> cudaError_t prefix_d(const PagedArgs &a, cudaStream_t s) {
    static const cudaError_t attr =
        cudaFuncSetAttribute(prefix_kernel<D, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
    if (attr != cudaSuccess) return attr;
    return launch_paged(prefix_kernel<D, DT>, dim3(unsigned(a.n_kv_heads * a.n_split * a.row_groups)), THREADS, Cfg<D>::SMEM, s, a);
}

}  // namespace

int prefix_ctas_per_sm(int dim) { return dim == 256 ? Cfg<256>::CTAS : Cfg<128>::CTAS; }

cudaError_t launch_paged_prefix(int dim, int dtype, const PagedArgs &a, cudaStream_t s) {
    if (a.n_split <= 0) return cudaSuccess;
    KVX_PAGED_DIM(prefix_d)
}

}  // namespace kvx
