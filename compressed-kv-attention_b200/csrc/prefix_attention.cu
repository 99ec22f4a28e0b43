// prefix_attention.cu -- attention of many query rows over one shared prefix, on the fifth-generation
// tensor cores.
//
// Every (sequence, query head) of a KV head is a row of one matrix: S = Q K^T and O += P V with up
// to 128 rows a CTA, so a piece of the prefix is read once for 128 rows.  One CTA takes one item:
// a KV head, 128 of its rows and a run of 64-token tiles; it leaves one partial state per row.
//
//  * The loader warps bring each K or V tile into a slot of a shared-memory ring in the layout the
//    tensor cores read (rows of 128 bytes, 16-byte pieces XOR-swizzled by the row; 64-byte rows at
//    D = 32).  From pages whose length is a multiple of 8 one warp does it with TMA: a tile is
//    64 / R boxes of R tokens (R the power of two, at most 64, that divides the page) a panel.  For
//    other lengths three warps copy row by row, 16 bytes a thread (64 x 32 heads of 128 behind 32768
//    tokens: 52 us by TMA, 62 by rows).
//  * One more warp issues the MMAs (one thread): S(i) = Q K(i)^T into one of two TMEM buffers, then O +=
//    P(i - 1) V(i - 1) with P read from TMEM (it replaces S there), so that S(i) is computed while the
//    softmax of tile i - 1 runs.  V is the N-major operand: the same rows as stored.
//  * Warps 0-3 do the softmax, a thread to a row: no shuffles.  The maximum that weights are
//    relative to is raised, and O rescaled in TMEM, only when some row's scores pass it by 2^8
//    (2^5 for FP16 weights), which is rare after the first tile; l and O share it, so it cancels.
//
// An XKV prefix takes the same kernel with other loader warps: each takes the tiles' 16-token groups
// in turn (every group's place, mode and escapes are in a table built with the prefix), brings a
// group's sign/mantissa bytes and residual codes into a staging slot of its own by two bulk copies,
// a few groups ahead, and rebuilds them into the ring's tile: BF16 words by byte permutes and one
// multiply-add a pair, escapes stored over them, rows past the block's end as zeros.  The blocks are
// decoded once for the item's 128 rows.
//
// What bounds it: per 64 tokens and 128 rows the SM's exponentials take 64 x 128 / 16 = 512 cycles, the
// MMAs at D = 128 about 600 (measured alone; S rereads Q for every 64 tokens) and the bytes from HBM
// 256 D / 23 (712 at D = 64, 1425 at D = 128, shared by all 128-row items of the head through L2).  On one
// B200, with the combine pass: 7 x 32 heads of 128 (28 rows) behind 131072 FP16 tokens 90 us, 6.0 TB/s, HBM;
// 64 x 32 heads (256 rows) behind 32768 BF16 tokens 51 us, 680 TFLOP/s, where copies alone take 38 and
// MMAs with softmax 37: two CTAs a SM overlap the rest; 32 x 32 heads behind 32731 coded tokens 53 us,
// where the decode alone takes 47 and the rest without it 44.
#include <cuda.h>

#include <utility>

#include "attention.cuh"
#include "paged_types.cuh"
#include "xkv_decode.cuh"

namespace kvx {
namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int TT = kPrefixTile;         // tokens per tile
constexpr int ROWS = kPrefixRows;       // query rows per item
constexpr int SW = 4;                   // softmax warps
constexpr uint32_t kDrainUs = 1000000;  // for copies and MMAs in flight, after a wait has run out

// Tensor maps of the K and V pools (LOAD_TMA).
struct alignas(64) PrefixMaps {
    CUtensorMap k, v;
};

// How the loader warps get the tiles: TMA boxes of whole page pieces, copies by row, or XKV blobs.
enum { LOAD_TMA, LOAD_ROWS, LOAD_XKV };

template <int D, int LOAD> struct Cfg {
    static constexpr bool XKV = LOAD == LOAD_XKV;
    // loader warps; an XKV group takes one about 2700 cycles at D = 128, hence as many as fit a SM's
    // registers and staging memory, with one CTA a SM (32 x 32 heads over 32731 tokens: two CTAs of three 75 us where this took 57)
    static constexpr int LW = LOAD == LOAD_TMA ? 1 : (LOAD == LOAD_ROWS ? 3 : (D == 256 ? 8 : 11));
    static constexpr int THREADS = 32 * (SW + LW + 1);
    static constexpr int ROWB = D >= 64 ? 128 : 64;         // bytes of a row of one panel of head dims
    static constexpr int SLOT = TT * D * 2;
    static constexpr int NSLOT = XKV ? (D == 32 ? 16 : (D == 64 ? 10 : (D == 128 ? 5 : 2))) : (D == 32 ? 12 : (D == 64 ? 10 : 5));
    static constexpr int LAG = (NSLOT - 1) / 2;                   // row copies: tiles in flight before one is announced
    static constexpr int PANELS = D >= 64 ? D / 64 : 1;
    static constexpr int CTAS = XKV || D == 256 ? 1 : 2;    // per SM
    static constexpr int O_Q = 0;
    static constexpr int O_RING = ROWS * D * 2;
    // staging slots of a loader warp (XKV): the group's table entry, 16 rows, their codes, each piece
    // landing 0-15 bytes past its 16-byte aligned start
    static constexpr int NSTAGE = XKV ? (D <= 64 ? 6 : (D == 128 ? 3 : 2)) : 0;
    static constexpr int S_ROWS = 32, S_CODES = S_ROWS + 16 * D + 32;
    static constexpr int STAGE = S_CODES + 8 * D + 32;
    static constexpr int O_STAGE = O_RING + NSLOT * SLOT;
    static constexpr int O_BAR = O_STAGE + LW * NSTAGE * STAGE;
    static constexpr int N_BAR = 2 * NSLOT + 10 + LW * NSTAGE;
    static constexpr int SMEM = O_BAR + 8 * N_BAR + 16;
    // arrivals that announce a tile: one of each loader warp, or one for each 16-token group
    static constexpr int ARRIVE = XKV ? TT / 16 : LW;  // (TMA: with the bytes)
    static constexpr int LDO = D + 4;                       // floats of a staged output row
    static constexpr int TMEM = D == 256 ? 512 : 256;       // columns: O at 0, S / P buffers at D, D + 64
    static constexpr uint64_t LAYOUT = D >= 64 ? 2 : 4;     // 128- / 64-byte swizzle
    static_assert(PANELS * (TT / 8) <= 32, "a lane for each TMA box");
    static_assert(XKV || LAG < NSLOT - 1 || LAG == 0, "the tile that frees the ring's next slot has been announced");
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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
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

// One TMA box global -> shared, completing its bytes on `bar`.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// 64 scores of this thread's row from TMEM, those from token `valid` on as -inf.
__device__ __forceinline__ void load_scores(uint32_t addr, int valid, uint32_t (&x)[64]) {
    uint32_t(&a)[32] = *reinterpret_cast<uint32_t(*)[32]>(&x[0]), (&b)[32] = *reinterpret_cast<uint32_t(*)[32]>(&x[32]);
    tmem_ld32(addr, a);
    tmem_ld32(addr + 32, b);
    tmem_wait_ld(a);
    tmem_wait_ld(b);
    if (valid < 64) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
            if (j >= valid) x[j] = 0xFF800000u;
    }
}

// Pairs of FP32 values in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Barriers of a CTA (8 bytes each): full and empty of every ring slot, these (S, P and PV of even and
// of odd tiles; QUIT: the MMAs issued before a wait ran out), then one for each staging slot.
enum { B_S0, B_S1, B_P0, B_P1, B_PV0, B_PV1, B_Q, B_END, B_DONE, B_QUIT, B_COUNT };

// One item.
struct Item {
    int head, first, n;   // KV head, first row, rows
    int tile0, tiles;
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
    x.tile0 = s * a.split_tiles;
    x.tiles = min(a.split_tiles, a.prefix_tiles - x.tile0);
    x.row0 = int64_t(x.head * a.n_split + s) * a.row_pad + x.first;
    return x;
}

// The ring's order for n tiles: K0, K1, V0, K2, V1, ..., K(n-1), V(n-2), V(n-1).
struct Ring {
    static __device__ __forceinline__ int k_item(int i) { return i == 0 ? 0 : 2 * i - 1; }
    static __device__ __forceinline__ int v_item(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }
    static __device__ __forceinline__ bool is_v(int q, int n) { return q == 2 * n - 1 || (q > 0 && (q & 1) == 0); }
    static __device__ __forceinline__ int tile(int q, int n) {
        return q == 0 ? 0 : (q == 2 * n - 1 ? n - 1 : (is_v(q, n) ? q / 2 - 1 : (q + 1) / 2));
    }
};

// Chunk steps of one 16-token group: rebuild them from the staged sections (coded modes) or the raw
// rows into the tile at `dst` (rows j0 .. j0 + 15), rows at or past n as zeros.
template <int D, int MODE>
__device__ __forceinline__ void decode_group(uint32_t stage_rows, uint32_t stage_codes, uint64_t raw, const Lay &ly,
                                             const uint32_t (&b7)[4], uint32_t dst, int j0, int n, int lane) {
    constexpr int C8 = D / 8, RPI = 32 / C8, STEPS = 16 / RPI, G = STEPS < 4 ? STEPS : 4;
    const int r0 = lane / C8, c8 = lane % C8;
#pragma unroll
    for (int k = 0; k < STEPS; k += G) {
        uint32_t W[G][MODE == 0 ? 5 : 3], X[G][2];
        if constexpr (MODE == 0) {
            // straight from the blob (raw blocks are rare): row sections start 0 or 2 bytes past a
            // word, and the word after the row's last is not read when it would be the blob's end
            const uint32_t *p = reinterpret_cast<const uint32_t *>(raw & ~uint64_t(3));
            const bool odd = (raw & 2u) != 0;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int r = r0 + RPI * (k + g);
#pragma unroll
                for (int i = 0; i < 5; ++i)
                    W[g][i] = r < n && (i < 4 || odd) ? __ldg(p + r * (D / 2) + 4 * c8 + i) : 0u;
            }
        } else {
            load_chunks<D, MODE, G, 0>(stage_rows + uint32_t(k * RPI * D), stage_codes + uint32_t(k * RPI * (D * MODE / 8)), W, X);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint32_t w[4];
            build_chunk<MODE>(ly, b7, W[g], X[g], w);
            const int r = r0 + RPI * (k + g);
            const bool in = r < n;
            sts_v4(dst + tile_off<D, TT>(j0 + r, c8), in ? w[0] : 0u, in ? w[1] : 0u, in ? w[2] : 0u, in ? w[3] : 0u);
        }
    }
}

template <int D, int DT, int LOAD>
__global__ void __launch_bounds__(Cfg<D, LOAD>::THREADS, Cfg<D, LOAD>::CTAS)
prefix_kernel(const PagedArgs a, const __grid_constant__ PrefixMaps maps) {
    using C = Cfg<D, LOAD>;
    constexpr bool XKV = C::XKV;
    constexpr int LW = C::LW;
    extern __shared__ __align__(1024) uint8_t smem[];
    volatile uint32_t *tmem_base = reinterpret_cast<volatile uint32_t *>(smem + C::O_BAR + 8 * C::N_BAR);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sb = smem_u32(smem);
    const uint32_t bars = sb + C::O_BAR;
    auto full = [&](int q) { return bars + 8u * uint32_t(q % C::NSLOT); };
    auto empty = [&](int q) { return bars + 8u * uint32_t(C::NSLOT + q % C::NSLOT); };
    auto bar = [&](int b) { return bars + 8u * uint32_t(2 * C::NSLOT + b); };
    const Item it = item_of(a, int(blockIdx.x));
    auto wait = [&](uint32_t b, int phase) -> bool {
        if (mbar_wait_bounded(b, uint32_t(phase & 1), uint32_t(a.wait_us))) return true;
        report(a.status, KVX_ERR_TIMEOUT, DERR_TIMEOUT);
        return false;
    };
    // copies and MMAs in flight end before the memory that they use goes away, whatever became of the waits
    auto drain = [&](uint32_t b, int phase) { mbar_wait_bounded(b, uint32_t(phase & 1), kDrainUs); };

    if (warp == SW + LW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bars + uint32_t(8 * C::N_BAR)),
                     "n"(C::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NSLOT; ++i) mbar_init(full(i), C::ARRIVE), mbar_init(empty(i), 1);
        for (int i = 0; i < LW * C::NSTAGE; ++i) mbar_init(bar(B_COUNT + i), 1);
        mbar_init(bar(B_S0), 1), mbar_init(bar(B_S1), 1), mbar_init(bar(B_P0), SW), mbar_init(bar(B_P1), SW);
        mbar_init(bar(B_PV0), 1), mbar_init(bar(B_PV1), 1), mbar_init(bar(B_Q), SW), mbar_init(bar(B_END), 1);
        mbar_init(bar(B_DONE), 1), mbar_init(bar(B_QUIT), 1);
        fence_mbar_init();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base;
    // what is above touches nothing of the grid before, which may still be running
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp >= SW && warp < SW + LW) {
        // ---- loads ----
        const int n_items = 2 * it.tiles;
        if constexpr (XKV) {
            // Loader warp w takes the 16-token groups w, w + LW, ... of the ring's items in order: each
            // tile's four arrivals come from whichever warps had them.
            constexpr int C8 = D / 8, NS = C::NSTAGE;
            const int w = warp - SW, c8 = lane % C8, r0 = lane / C8;
            const int total = n_items * (TT / 16), mine = (total - w + LW - 1) / LW;
            const uint32_t stages = sb + uint32_t(C::O_STAGE + w * NS * C::STAGE);
            const XkvGroup *groups = a.xkv.groups + int64_t(it.head) * a.xkv.head_tiles * (2 * (TT / 16));
            auto entry = [&](int k) -> const uint4 * {
                const int id = w + LW * k, q = id / (TT / 16), tile = it.tile0 + Ring::tile(q, it.tiles);
                return reinterpret_cast<const uint4 *>(groups + (2 * tile + (Ring::is_v(q, it.tiles) ? 1 : 0)) * (TT / 16) + id % (TT / 16));
            };
            auto staged = [&](int k) { return bar(B_COUNT + w * NS + k % NS); };
            // group k into its staging slot: the table entry, and the copies of a coded group (lane 0 the
            // rows, lane 1 the codes)
            auto issue = [&](int k, const uint4 &e0, const uint4 &e1) {
                const uint32_t slot = stages + uint32_t(k % NS * C::STAGE);
                const uint32_t len = lane == 0 ? e1.z & 0xFFFFu : e1.z >> 16;
                if (lane == 0) {
                    sts_v4(slot, e0.x, e0.y, e0.z, e0.w);
                    sts_v4(slot + 16, e1.x, e1.y, e1.z, e1.w);
                    mbar_arrive_expect_tx(staged(k), (e1.z & 0xFFFFu) + (e1.z >> 16));
                }
                if (lane < 2 && len != 0u) {
                    const uint64_t at = lane == 0 ? (uint64_t(e0.y) << 32) | e0.x : (uint64_t(e0.w) << 32) | e0.z;
                    bulk_g2s(slot + (lane == 0 ? C::S_ROWS : C::S_CODES), reinterpret_cast<const void *>(at), len, staged(k));
                }
            };
            uint4 e0 = make_uint4(0u, 0u, 0u, 0u), e1 = e0;
            int issued = 0;
            for (; issued < NS && issued < mine; ++issued) {
                const uint4 *p = entry(issued);
                issue(issued, __ldg(p), __ldg(p + 1));
            }
            if (issued < mine) e0 = __ldg(entry(issued)), e1 = __ldg(entry(issued) + 1);
            __syncwarp();
            // what a group needs from global memory besides its copies, fetched a group ahead: the
            // lane's merge words and escape entry
            XkvGroup next;
            uint4 b7n = make_uint4(0u, 0u, 0u, 0u);
            uint32_t escn = 0;
            auto fetch = [&](int k) {
                const uint32_t slot = stages + uint32_t(k % NS * C::STAGE);
                uint4 h0, h1;
                lds_v4(slot, h0.x, h0.y, h0.z, h0.w);
                lds_v4(slot + 16, h1.x, h1.y, h1.z, h1.w);
                next.rows = (uint64_t(h0.y) << 32) | h0.x;
                next.esc = h1.x, next.b7 = h1.y, next.bits = h1.w;
                if (next.mode() != 0) b7n = __ldg(reinterpret_cast<const uint4 *>(a.xkv.b7 + next.b7) + c8);
                if (lane < next.n_esc()) escn = __ldg(a.xkv.esc + next.esc + lane);
            };
            if (mine > 0) fetch(0);
            bool ok = true;
            int k = 0;
            for (; k < mine; ++k) {
                const int id = w + LW * k, q = id / (TT / 16), j0 = 16 * (id % (TT / 16));
                const XkvGroup grp = next;
                const uint32_t b7[4] = {b7n.x, b7n.y, b7n.z, b7n.w}, ent = escn;
                if (k + 1 < mine) fetch(k + 1);
                if (q >= C::NSLOT) ok = __all_sync(FULL, wait(empty(q), q / C::NSLOT - 1));
                if (ok) ok = __all_sync(FULL, wait(staged(k), k / NS));
                if (!ok) break;
                const int n_esc = grp.n_esc(), mode = grp.mode(), n = grp.n();
                const uint32_t slot = stages + uint32_t(k % NS * C::STAGE);
                const uint32_t dst = sb + uint32_t(C::O_RING + (q % C::NSLOT) * C::SLOT);
                const Lay ly = make_lay<D>(grp.row_off(), grp.code_off(), mode, c8, false, C::S_CODES - C::S_ROWS);
                const uint32_t sr = slot + C::S_ROWS + ly.rows + uint32_t(r0 * D), sc = slot + C::S_ROWS + ly.codes;
                if (mode == 4) decode_group<D, 4>(sr, sc + uint32_t(r0 * (D / 2)), 0, ly, b7, dst, j0, n, lane);
                else if (mode == 2) decode_group<D, 2>(sr, sc + uint32_t(r0 * (D / 4)), 0, ly, b7, dst, j0, n, lane);
                else if (mode == 3) decode_group<D, 3>(sr, sc + uint32_t(r0 * (D * 3 / 8)), 0, ly, b7, dst, j0, n, lane);
                else decode_group<D, 0>(0, 0, grp.rows, ly, b7, dst, j0, n, lane);
                __syncwarp();
                // escapes: the entry's element by its byte in a 16-row tile (swizzled like this one's rows)
                for (int i = lane; i < n_esc; i += 32) {
                    const uint32_t e = i == lane ? ent : __ldg(a.xkv.esc + grp.esc + i);
                    const uint32_t at = e & 0xFFFEu, r = at / (2 * D), in_row = at % (2 * D);
                    if (int(r) < n)
                        sts_u16(dst + (in_row / C::ROWB) * (TT * C::ROWB) + (uint32_t(j0) + r) * C::ROWB + in_row % C::ROWB, e >> 16);
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(full(q));
                if (issued < mine) {
                    issue(issued, e0, e1);
                    ++issued;
                    if (issued < mine) e0 = __ldg(entry(issued)), e1 = __ldg(entry(issued) + 1);
                    __syncwarp();
                }
            }
            for (; k < issued; ++k) drain(staged(k), k / NS);  // (none are left where no wait ran out)
        } else if constexpr (LOAD == LOAD_TMA) {
            // Lane i loads box i of a tile: box_tokens tokens of one panel of 64 head dims.  pages of the
            // latest K tile, of the one before it (V follows a tile behind) and of the next; -1: no
            // tokens there.
            const int box = a.box_tokens, per = TT / box;
            const int p = lane / per, t = (lane - p * per) * box;
            const uint32_t at = uint32_t(p * (TT * C::ROWB) + t * C::ROWB), bytes = uint32_t(box * C::ROWB);
            int place_k = 0, place_before = 0, place_next = 0;
            // (nothing looks at the entry before the next K tile: its load is not waited for here)
            auto look_up = [&](int tile, int &place) -> int32_t {
                const int tok = (it.tile0 + tile) * TT + t;
                place = -1;
                if (tile >= it.tiles || p >= C::PANELS || tok >= a.prefix_len) return 0;
                int64_t i;
                a.pool.split.at(tok, i, place);
                return __ldg(a.prefix_table + i);
            };
            int32_t pg_k = 0, pg_before = 0, pg_next = look_up(0, place_next);
            bool ok = true;
            int q = 0;
            for (; q < n_items; ++q) {
                const bool is_v = Ring::is_v(q, it.tiles);
                const int tile = Ring::tile(q, it.tiles);
                if (!is_v) {
                    pg_before = pg_k, place_before = place_k;
                    pg_k = pg_next, place_k = place_next;
                    pg_next = look_up(tile + 1, place_next);
                }
                if (q >= C::NSLOT) ok = __all_sync(FULL, wait(empty(q), q / C::NSLOT - 1));
                if (!ok) break;
                const bool before = is_v && q < n_items - 1;
                const int32_t pg = before ? pg_before : pg_k;
                const int place = before ? place_before : place_k;
                bool live = place >= 0;
                if (live && unsigned(pg) >= unsigned(a.pool.n_pages)) {
                    report(a.status, KVX_ERR_RUNTIME, DERR_PAGE);
                    live = false;
                }
                const uint32_t dst = sb + uint32_t(C::O_RING + (q % C::NSLOT) * C::SLOT);
                // V rows past the prefix's end meet weights of 0 and must be finite: that tile's boxes
                // are waited for here and the rows zeroed before the tile is announced
                const int valid = a.prefix_len - (it.tile0 + tile) * TT;
                const bool ends = is_v && valid < TT;
                const uint32_t to = ends ? bar(B_END) : full(q);
                const uint32_t boxes = uint32_t(__popc(__ballot_sync(FULL, live)));
                if (lane == 0) mbar_arrive_expect_tx(to, boxes * bytes);
                __syncwarp();
                if (live)
                    tma_load(dst + at, is_v ? &maps.v : &maps.k, p * 64, a.heads_inside ? it.head : place,
                             a.heads_inside ? place : it.head, pg, to);
                if (ends) {
                    ok = __all_sync(FULL, wait(to, 0));
                    if (!ok) {
                        drain(to, 0);
                        break;
                    }
                    for (int i = lane; i < (TT - valid) * (D / 8); i += 32)
                        sts_v4(dst + tile_off<D, TT>(valid + i / (D / 8), i % (D / 8)), 0u, 0u, 0u, 0u);
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(q));
                }
            }
            // (the MMA warp, which waits for the boxes, may have given up)
            for (int i = max(0, q - C::NSLOT); i < q; ++i) drain(full(i), i / C::NSLOT);
        } else {
        // Loader warp w copies rows w, w + LW, ... of every tile: lane k holds the offsets of rows w + LW k
        // and w + LW (k + 32) (-1: no such token), looked up a tile ahead of their use.
        constexpr int CH = D / 8, RPS = 32 / CH;              // pieces a row, rows a step
        constexpr int MINE = (TT + LW - 1) / LW, STEPS = (MINE + RPS - 1) / RPS, H = (MINE + 31) / 32;
        const int w = warp - SW, c = lane % CH;
        const int64_t head = int64_t(it.head) * a.pool.head_stride + 8 * c;
        // (nothing looks at the entries before the next K tile: their loads are not waited for here)
        int32_t page_next[H];
        int place_next[H];
        auto look_up = [&](int tile) {
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int r = w + LW * (lane + 32 * h), tok = (it.tile0 + tile) * TT + r;
                place_next[h] = -1, page_next[h] = 0;
                if (r < TT && tok < a.prefix_len && tile < it.tiles) {
                    int64_t i;
                    a.pool.split.at(tok, i, place_next[h]);
                    page_next[h] = __ldg(a.prefix_table + i);
                }
            }
        };
        auto announce = [&](int i) {
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(full(i));
        };
        // rows of the latest K tile and of the one before it (V follows a tile behind)
        int64_t r_k[H], r_before[H];
        look_up(0);
#pragma unroll
        for (int h = 0; h < H; ++h) r_k[h] = r_before[h] = -1;
        bool ok = true;
        int q = 0;
        for (; q < n_items; ++q) {
            const bool is_v = Ring::is_v(q, it.tiles);
            if (!is_v) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    r_before[h] = r_k[h];
                    r_k[h] = -1;
                    if (place_next[h] < 0) continue;
                    if (unsigned(page_next[h]) < unsigned(a.pool.n_pages))
                        r_k[h] = int64_t(page_next[h]) * a.pool.page_stride + int64_t(place_next[h]) * a.pool.token_stride;
                    else report(a.status, KVX_ERR_RUNTIME, DERR_PAGE);
                }
                look_up(Ring::tile(q, it.tiles) + 1);
            }
            if (q >= C::NSLOT) ok = __all_sync(FULL, wait(empty(q), q / C::NSLOT - 1));
            if (!ok) break;
            const uint16_t *src = (is_v ? a.pool.v : a.pool.k) + head;
            const uint32_t dst = sb + uint32_t(C::O_RING + (q % C::NSLOT) * C::SLOT);
            const bool before = is_v && q < n_items - 1;
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                const int k = j * RPS + lane / CH, r = w + LW * k;
                const int h = j * RPS / 32;
                const int64_t o = __shfl_sync(FULL, before ? r_before[h] : r_k[h], k & 31);
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
        }
    } else if (warp == SW + LW) {
        // ---- MMAs ----
        if (lane == 0) {
            constexpr uint32_t qk = instr_desc<DT>(TT, false), pv = instr_desc<DT>(D, true);
            constexpr uint32_t K8 = 8 * C::ROWB;  // bytes of 8 rows
            // descriptors of a tile are its base's plus steps of the start address
            const uint64_t q0 = smem_desc(sb + C::O_Q, 16, K8, C::LAYOUT), k0 = smem_desc(sb + C::O_RING, 16, K8, C::LAYOUT),
                           v0 = smem_desc(sb + C::O_RING, TT * C::ROWB, K8, C::LAYOUT);
            bool ok = wait(bar(B_Q), 0) && a.wait_us > 0;  // (0: no S is begun, so that every row's wait runs out)
            for (int i = 0; ok && i <= it.tiles; ++i) {
                if (i < it.tiles) {
                    const int x = Ring::k_item(i);
                    ok = wait(full(x), x / C::NSLOT);
                    if (!ok) break;
                    fence_after();
                    const uint64_t kk = k0 + uint32_t(x % C::NSLOT) * uint32_t(C::SLOT / 16);
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        const uint32_t p = uint32_t(s / (C::ROWB / 32)), o = uint32_t(s % (C::ROWB / 32)) * 32;
                        mma_ss(tm + D + (i & 1) * TT, q0 + (p * (ROWS * C::ROWB) + o) / 16, kk + (p * (TT * C::ROWB) + o) / 16, qk,
                               s > 0);
                    }
                    mma_commit(bar(B_S0 + (i & 1)));
                    mma_commit(empty(x));
                }
                if (i > 0) {
                    const int j = i - 1, x = Ring::v_item(j, it.tiles);
                    ok = wait(full(x), x / C::NSLOT) && wait(bar(B_P0 + (j & 1)), j >> 1);
                    if (!ok) break;
                    fence_after();
                    const uint64_t vv = v0 + uint32_t(x % C::NSLOT) * uint32_t(C::SLOT / 16);
#pragma unroll
                    for (int s = 0; s < TT / 16; ++s)
                        mma_ts(tm, tm + D + (j & 1) * TT + 8 * s, vv + 2 * s * K8 / 16, pv, j > 0 || s > 0);
                    mma_commit(bar(B_PV0 + (j & 1)));
                    mma_commit(empty(x));
                    if (j == it.tiles - 1) mma_commit(bar(B_DONE));
                }
            }
            if (!ok) mma_commit(bar(B_QUIT));
            drain(bar(ok ? B_DONE : B_QUIT), 0);
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
            int valid = a.prefix_len - (it.tile0 + i) * TT;  // tokens of the tile
            if constexpr (XKV)
                valid = __ldg(a.xkv.tile_tokens + int64_t(it.head) * a.xkv.head_tiles + it.tile0 + i);
            ok = __all_sync(FULL, wait(bar(B_S0 + (i & 1)), i >> 1));
            if (!ok) break;
            fence_after();
            if (live) {
                const uint32_t st = tm + lanes + uint32_t(D + (i & 1) * TT);
                uint32_t x[64];
                load_scores(st, valid, x);
                float y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    y[k] = __uint_as_float(x[k]);
#pragma unroll
                    for (int j = 4; j + 4 < 64; j += 8) y[k] = max3(y[k], __uint_as_float(x[j + k]), __uint_as_float(x[j + 4 + k]));
                    y[k] = fmaxf(y[k], __uint_as_float(x[60 + k]));
                }
                float mx = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
                mx *= a.scale_log2;
                if (__any_sync(FULL, mx > m + kGrow || (m == -INFINITY && mx > m))) {
                    const float mn = fmaxf(m, mx);
                    const float al = mn == -INFINITY ? 1.f : exp2_sfu(m - mn);
                    m = mn;
                    l *= al;
                    if (i > 0) {
                        // O is complete up to tile i - 1, and the next PV waits for this warp
                        ok = __all_sync(FULL, wait(bar(B_PV0 + ((i - 1) & 1)), (i - 1) >> 1));
                        if (!ok) break;
                        fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += 16) {  // (16 columns: the scores stay in registers)
                            uint32_t o[16];
                            tmem_ld16(tm + lanes + c, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * al);
                            tmem_st16(tm + lanes + c, o);
                        }
                    }
                }
                const float mu = m == -INFINITY ? 0.f : m - Elem<DT>::kBias;
                const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), mu2 = pair(-mu, -mu);
                uint64_t sum[2] = {pair(l, 0.f), pair(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t p[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float u, v;
                        unpair(fma2(pair(__uint_as_float(x[32 * h + 2 * j]), __uint_as_float(x[32 * h + 2 * j + 1])), scale2, mu2), u, v);
                        u = exp2_sfu(u), v = exp2_sfu(v);
                        sum[j & 1] = add2(sum[j & 1], pair(u, v));
                        p[j] = Elem<DT>::pack(u, v);
                    }
                    tmem_st16(st + 16 * h, p);
                }
                float u, v;
                unpair(add2(sum[0], sum[1]), u, v);
                l = u + v;
                tmem_wait_st();
            }
            // PV(i - 2) completed before S(i) did; its barrier is waited for all the same, before the arrival
            // that lets PV(i) complete: a phase later its parity would not tell one from the other.  (That
            // PV(i - 1) is not waited for lets two tiles' round trips between these warps and the MMA warp
            // overlap.)
            if (i > 1) ok = __all_sync(FULL, wait(bar(B_PV0 + (i & 1)), (i - 2) >> 1));
            if (!ok) break;
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_P0 + (i & 1)));
        }
        if (ok) ok = __all_sync(FULL, wait(bar(B_DONE), 0));
        const int n = min(32, it.n - 32 * warp);  // rows of this warp
        // after a wait that ran out the rows' outputs become NaN (what an earlier call left there is no part of them)
        if (!ok && lane < n) a.ml[it.row0 + 32 * warp + lane] = make_float2(-INFINITY, __int_as_float(0x7FFFFFFF));
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

template <int D, int DT, int LOAD>
cudaError_t prefix_launch(const PagedArgs &a, const PrefixMaps &maps, cudaStream_t s) {
    using C = Cfg<D, LOAD>;
    return launch_paged(prefix_kernel<D, DT, LOAD>, dim3(unsigned(a.n_kv_heads * a.n_split * a.row_groups)), C::THREADS, C::SMEM, s, a, maps);
}

// The driver's tensor map encoder (found at run time: the library links no libcuda).
using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn tensor_map_encoder() {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        cudaGetLastError();
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Maps of one layer's pools with boxes of a.box_tokens tokens of 64 (32) head dims; the nearer of
// tokens and heads inside (a.heads_inside).  false: the driver takes no such map.
bool encode_maps(int dim, int dtype, PagedArgs &a, PrefixMaps &maps) {
    const EncodeFn encode = tensor_map_encoder();
    if (encode == nullptr) return false;
    const PoolDev &p = a.pool;
    // (a dimension of one element has no stride of its own: any will do)
    const int64_t row = int64_t(dim) * 2;
    const int64_t token = p.split.tokens > 1 ? p.token_stride * 2 : row, head = a.n_kv_heads > 1 ? p.head_stride * 2 : row,
                  page = p.n_pages > 1 ? p.page_stride * 2 : row;
    a.heads_inside = a.n_kv_heads > 1 && p.head_stride < p.token_stride;
    if (token <= 0 || head <= 0 || page <= 0) return false;
    const cuuint64_t tokens = cuuint64_t(p.split.tokens), heads = cuuint64_t(a.n_kv_heads), pages = cuuint64_t(p.n_pages);
    const cuuint32_t b = cuuint32_t(a.box_tokens), inner = dim >= 64 ? 64u : 32u;
    cuuint64_t dims[4] = {cuuint64_t(dim), tokens, heads, pages}, strides[3] = {cuuint64_t(token), cuuint64_t(head), cuuint64_t(page)};
    cuuint32_t box[4] = {inner, b, 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
    if (a.heads_inside) {
        std::swap(dims[1], dims[2]);
        std::swap(strides[0], strides[1]);
        std::swap(box[1], box[2]);
    }
    const CUtensorMapDataType type = dtype == KVX_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUtensorMapSwizzle swizzle = dim >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    for (int T = 0; T < 2; ++T)
        if (encode(T ? &maps.v : &maps.k, type, 4, T ? p.v : p.k, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

template <int D, int DT> cudaError_t prefix_d(const PagedArgs &args, cudaStream_t s) {
    PagedArgs a = args;
    PrefixMaps maps{};
    if constexpr (DT == KVX_DTYPE_BF16)
        if (a.xkv.tiles > 0) return prefix_launch<D, DT, LOAD_XKV>(a, maps, s);
    // boxes of fewer than 8 tokens would not fill a swizzle pattern
    for (a.box_tokens = kPrefixTile; a.pool.split.tokens % a.box_tokens != 0;) a.box_tokens >>= 1;
    if (a.box_tokens >= 8 && encode_maps(D, DT, a, maps)) return prefix_launch<D, DT, LOAD_TMA>(a, maps, s);
    return prefix_launch<D, DT, LOAD_ROWS>(a, maps, s);
}

template <int D, int DT> cudaError_t prepare_d() {
    cudaError_t e = allow_smem(prefix_kernel<D, DT, LOAD_TMA>, Cfg<D, LOAD_TMA>::SMEM);
    if (e == cudaSuccess) e = allow_smem(prefix_kernel<D, DT, LOAD_ROWS>, Cfg<D, LOAD_ROWS>::SMEM);
    if constexpr (DT == KVX_DTYPE_BF16)
        if (e == cudaSuccess) e = allow_smem(prefix_kernel<D, DT, LOAD_XKV>, Cfg<D, LOAD_XKV>::SMEM);
    return e;
}

// One thread per (flat block, tile): its groups and its token count.
__global__ void xkv_groups_kernel(const BlockDesc *desc, int64_t n, int tpb, int dim, XkvGroup *groups, uint8_t *tokens) {
    const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n * tpb) return;
    const int64_t b = i / tpb;
    const int sub = int(i - b * tpb);
    const BlockDesc &d = desc[b];
    const int left = int(d.valid) - sub * TT;
    tokens[i] = uint8_t(left < 0 ? 0 : (left < TT ? left : TT));
    for (int T = 0; T < 2; ++T) {
        const uint64_t blk = T ? d.v : d.k;
        const int mode = T ? d.v_mode : d.k_mode, nesc = T ? d.v_nesc : d.k_nesc;
        for (int j = 0; j < TT / 16; ++j) {
            const int g16 = sub * (TT / 16) + j, t0 = 16 * g16;
            XkvGroup g{};
            const int m = int(d.valid) - t0;
            const uint32_t n_tok = uint32_t(m < 0 ? 0 : (m < 16 ? m : 16));
            uint32_t n_esc = 0, row_off = 0, code_off = 0;
            g.b7 = uint32_t(d.b7_block) * uint32_t(dim) + uint32_t(T * (dim / 2));
            if (n_tok > 0 && mode == 0) {
                g.rows = blk + kHeaderBytes + uint64_t(t0) * dim * 2;
                row_off = uint32_t(g.rows & 2u);
            } else if (n_tok > 0) {
                const uint64_t rows = blk + kHeaderBytes + dim + uint64_t(t0) * dim;
                const uint64_t codes = blk + kHeaderBytes + dim + uint64_t(d.n_tok) * dim + uint64_t(t0) * dim * mode / 8;
                row_off = uint32_t(rows & 15u), code_off = uint32_t(codes & 15u);
                g.rows = rows - row_off, g.codes = codes - code_off;
                g.n_rows = uint16_t((row_off + n_tok * dim + 15u) & ~15u);
                g.n_codes = uint16_t((code_off + n_tok * dim * mode / 8 + 15u) & ~15u);
                if (nesc != 0) {
                    const int e0 = g16 == 0 ? 0 : d.em[T][g16 - 1], e1 = d.em[T][g16];
                    g.esc = (T ? d.v_rec : d.k_rec) + uint32_t(kEscRecHead + e0);
                    n_esc = uint32_t(e1 - e0);
                }
            }
            g.bits = n_esc | (n_tok << 13) | (uint32_t(mode) << 18) | (row_off << 20) | (code_off << 23);
            groups[(i * 2 + T) * (TT / 16) + j] = g;
        }
    }
}

}  // namespace

int prefix_ctas_per_sm(int dim, bool coded) { return coded || dim == 256 ? Cfg<256, LOAD_TMA>::CTAS : Cfg<128, LOAD_TMA>::CTAS; }

cudaError_t launch_xkv_groups(const BlockDesc *desc, int64_t n_blocks, int tiles_per_block, int dim, XkvGroup *groups,
                              uint8_t *tile_tokens, cudaStream_t s) {
    const int64_t n = n_blocks * tiles_per_block;
    if (n <= 0) return cudaSuccess;
    xkv_groups_kernel<<<unsigned((n + 127) / 128), 128, 0, s>>>(desc, n_blocks, tiles_per_block, dim, groups, tile_tokens);
    return cudaGetLastError();
}

cudaError_t prepare_paged_prefix(int dim, int dtype) { KVX_PAGED_DIM(prepare_d) }

cudaError_t launch_paged_prefix(int dim, int dtype, const PagedArgs &a, cudaStream_t s) {
    if (a.n_split <= 0) return cudaSuccess;
    KVX_PAGED_DIM(prefix_d, a, s)
}

}  // namespace kvx
