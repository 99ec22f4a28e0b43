// paged_stream.cu -- single-token attention over paged keys and values, up to 8 query rows at a
// time, and the combine pass that folds every row's partial states.
//
// One CTA takes one item: up to 8 query rows and a run of tokens of one KV head, either a chunk of
// one sequence's own pages or (batches of few rows) a piece of the shared prefix.  Its 8 warps take
// the run's 16-token tiles in turn, each with its own online softmax, and join their states in
// shared memory; the CTA leaves one partial state per row.
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
constexpr int NW = 8;  // warps per CTA

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

// An item: query rows and a run of tokens.
struct Item {
    const int32_t *table;
    int64_t row0;       // first partial row
    int t0, t1;         // tokens
    int first, n;       // rows first .. first + n - 1 of the head's (sequence, g) list
    int head;           // KV head
};

__device__ __forceinline__ bool item_of(const PagedArgs &a, int i, Item &x) {
    if (i < a.prefix_items) {
        const int rg = i % a.row_groups;
        i /= a.row_groups;
        const int s = i % a.n_split;
        x.head = i / a.n_split;
        x.table = a.prefix_table;
        x.t0 = s * a.split_tokens;
        x.t1 = min(a.prefix_len, x.t0 + a.split_tokens);
        x.first = 8 * rg;
        x.n = min(8, a.batch * a.group - x.first);
        x.row0 = int64_t(x.head * a.n_split + s) * a.row_pad + x.first;
        return true;
    }
    i -= a.prefix_items;
    const int qg = i % a.q_groups;
    i /= a.q_groups;
    const int c = i % a.n_chunk;
    i /= a.n_chunk;
    x.head = i % a.n_kv_heads;
    const int b = i / a.n_kv_heads;
    x.t0 = c * a.chunk_tokens;
    x.t1 = min(tail_len(a, b), x.t0 + a.chunk_tokens);
    x.table = a.table + int64_t(b) * a.table_stride;
    x.first = b * a.group + 8 * qg;
    x.n = min(8, a.group - 8 * qg);
    x.row0 = a.tail_base + (int64_t(b * a.n_kv_heads + x.head) * a.n_chunk + c) * a.group + 8 * qg;
    return x.t0 < x.t1;  // a chunk past the sequence's end has no state; the combine does not look
}

template <int D> constexpr int stream_smem() { return NW * 8 * D * 4; }

template <int D, int DT>
__global__ void __launch_bounds__(NW * 32, D <= 128 ? 2 : 1) stream_kernel(const PagedArgs a) {
    constexpr int KJ = D / 32;                 // 32-dim pieces of a K row
    constexpr int VI = D >= 64 ? D / 64 : 1;   // pieces of a V row
    constexpr int VW = D >= 64 ? 4 : 2;        // words a lane loads of each
    extern __shared__ float sacc[];            // [NW][8][D]
    __shared__ float2 sml[NW][8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Item it;
    if (!item_of(a, int(blockIdx.x), it)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;

    // Q rows as A fragments
    uint4 qf[KJ];
    {
        const int r = it.first + (g < it.n ? g : 0), b = r / a.group;
        const uint16_t *q = a.q + int64_t(b) * a.q_token + int64_t(it.head * a.group + r - b * a.group) * a.q_head + 8 * t;
#pragma unroll
        for (int j = 0; j < KJ; ++j) qf[j] = g < it.n ? load16(q + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
    }
    const uint16_t *kb = a.pool.k + int64_t(it.head) * a.pool.head_stride + 8 * t;
    const uint16_t *vb = a.pool.v + int64_t(it.head) * a.pool.head_stride + 2 * VW * g;

    float acc[VI * VW][4];
#pragma unroll
    for (int i = 0; i < VI * VW; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    float m = -INFINITY, l = 0.f;

    // lanes 0-15 look up the rows of the next tile's tokens, a tile ahead (-1: no such token)
    auto rows_of = [&](int tile) -> int64_t {
        const int tok = tile + (lane & 15);
        return tile < it.t1 && tok < it.t1 ? page_row(a.pool, it.table, tok, a.status) : -1;
    };
    int64_t nxt = rows_of(it.t0 + 16 * warp);
    for (int tile = it.t0 + 16 * warp; tile < it.t1; tile += 16 * NW) {
        const int64_t row = nxt;
        uint4 kf[2][KJ];
        bool live[2][2];  // tokens 8 n + 2 t, 8 n + 2 t + 1
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int64_t r = __shfl_sync(FULL, row, 8 * n + g);
#pragma unroll
            for (int j = 0; j < KJ; ++j) kf[n][j] = r >= 0 ? load16(kb + r + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
        }
        uint32_t vf[4][VI][VW];
        auto load_v = [&]() {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t r = __shfl_sync(FULL, row, 2 * t + (k & 1) + 8 * (k >> 1));
                live[k >> 1][k & 1] = r >= 0;
#pragma unroll
                for (int i = 0; i < VI; ++i) {
                    if constexpr (VW == 4) {
                        const uint4 v = r >= 0 ? load16(vb + r + 64 * i) : make_uint4(0u, 0u, 0u, 0u);
                        vf[k][i][0] = v.x, vf[k][i][1] = v.y, vf[k][i][2] = v.z, vf[k][i][3] = v.w;
                    } else {
                        const uint2 v = r >= 0 ? load8(vb + r) : make_uint2(0u, 0u);
                        vf[k][i][0] = v.x, vf[k][i][1] = v.y;
                    }
                }
            }
        };
        if constexpr (D <= 128) load_v();  // (at 256 the registers hold one of K and V at a time)
        nxt = rows_of(tile + 16 * NW);

        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                mma16<DT>(s[n], qf[j].x, 0u, qf[j].y, 0u, kf[n][j].x, kf[n][j].y);
                mma16<DT>(s[n], qf[j].z, 0u, qf[j].w, 0u, kf[n][j].z, kf[n][j].w);
            }
        }
        if constexpr (D > 128) load_v();
        // online softmax of query g: this lane has 4 of the 16 tokens
        float x[2][2];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[n][e] = live[n][e] ? s[n][e] * a.scale_log2 : -INFINITY;
        float mx = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1]));
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
        float p[2][2];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) p[n][e] = exp2_sfu(x[n][e] - mu), l += p[n][e];
        const uint32_t b0 = Elem<DT>::pack(p[0][0], p[0][1]), b1 = Elem<DT>::pack(p[1][0], p[1][1]);
#pragma unroll
        for (int i = 0; i < VI; ++i)
#pragma unroll
            for (int w = 0; w < VW; ++w)
                mma16<DT>(acc[i * VW + w], prmt(vf[0][i][w], vf[1][i][w], 0x5410u), prmt(vf[0][i][w], vf[1][i][w], 0x7632u),
                          prmt(vf[2][i][w], vf[3][i][w], 0x5410u), prmt(vf[2][i][w], vf[3][i][w], 0x7632u), b0, b1);
    }

    // join the warps' states
    l += __shfl_xor_sync(FULL, l, 1);
    l += __shfl_xor_sync(FULL, l, 2);
    if (t == 0) sml[warp][g] = make_float2(m, l);
    __syncthreads();
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[w][g].x);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float2 z = sml[w][g];
        L += z.x == -INFINITY ? z.y * 0.f : z.y * exp2_sfu(z.x - M);  // (l is 0, or NaN, without a maximum)
    }
    const float f = m == -INFINITY ? 0.f : exp2_sfu(m - M);
    const float f0 = __shfl_sync(FULL, f, 8 * t), f1 = __shfl_sync(FULL, f, 8 * t + 4);
#pragma unroll
    for (int i = 0; i < VI; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            const float(&c)[4] = acc[i * VW + w];
            const int d = 64 * i + 2 * VW * g + 2 * w;
            float *o = sacc + (warp * 8 + 2 * t) * D + d;
            *reinterpret_cast<float2 *>(o) = make_float2(c[0] * f0, c[2] * f0);
            *reinterpret_cast<float2 *>(o + D) = make_float2(c[1] * f1, c[3] * f1);
        }
    __syncthreads();
    if (warp == 0 && t == 0 && g < it.n)
        a.ml[it.row0 + g] = make_float2(M == -INFINITY ? M : M - Elem<DT>::kBias, L);
    for (int i = threadIdx.x; i < it.n * (D / 4); i += NW * 32) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 u = reinterpret_cast<const float4 *>(sacc + w * 8 * D)[i];
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        reinterpret_cast<float4 *>(a.acc + it.row0 * D)[i] = v;
    }
}

// Folds the partial states of one (sequence, head): M = max m_i, l = sum l_i 2^(m_i - M), out =
// (sum acc_i 2^(m_i - M)) / l.  One CTA per row, its warps take the parts in turn; sums run in a
// fixed order.
template <int D, int DT>
__global__ void __launch_bounds__(512) combine_kernel(const PagedArgs a) {
    constexpr int V = D / 32;  // values per lane
    __shared__ float sacc[16][D];
    __shared__ float sl[16];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = blockIdx.y, h = blockIdx.x, head = h / a.group, gi = h - head * a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int np = a.n_split;
    const int nt = a.n_chunk > 0 ? (tail_len(a, b) + a.chunk_tokens - 1) / a.chunk_tokens : 0;
    const int64_t prow = int64_t(head) * a.n_split * a.row_pad + b * a.group + gi;
    const int64_t trow = a.tail_base + int64_t(b * a.n_kv_heads + head) * a.n_chunk * a.group + gi;
    auto row = [&](int i) -> int64_t {
        return i < np ? prow + int64_t(i) * a.row_pad : trow + int64_t(i - np) * a.group;
    };
    float M = -INFINITY;
    for (int i = lane; i < np + nt; i += 32) M = fmaxf(M, a.ml[row(i)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(FULL, M, o));
    float o[V], l = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll 4
    for (int i = warp; i < np + nt; i += nw) {
        const int64_t r = row(i);
        const float2 z = a.ml[r];
        const float w = z.x == -INFINITY ? 0.f : exp2_sfu(z.x - M);
        l += z.y * w;
        const float *p = a.acc + r * D + V * lane;
        if (z.x != -INFINITY || z.y != z.y) {
            if constexpr (V == 1) o[0] += w * p[0];
            else if constexpr (V == 2) {
                const float2 u = *reinterpret_cast<const float2 *>(p);
                o[0] += w * u.x, o[1] += w * u.y;
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const float4 u = *reinterpret_cast<const float4 *>(p + j);
                    o[j] += w * u.x, o[j + 1] += w * u.y, o[j + 2] += w * u.z, o[j + 3] += w * u.w;
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sacc[warp][V * lane + j] = o[j];
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    l = 0.f;
    for (int w = 0; w < nw; ++w) l += sl[w];
    uint16_t *out = a.out + int64_t(b) * a.out_token + int64_t(h) * a.out_head;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float v = 0.f;
        for (int w = 0; w < nw; ++w) v += sacc[w][d];
        out[d] = Elem<DT>::one(l == 0.f ? 0.f : v / l);
    }
    if (threadIdx.x == 0 && a.lse != nullptr)
        a.lse[int64_t(b) * a.n_q_heads + h] = l == 0.f ? -INFINITY : M * kPagedLn2 + logf(l);
}

template <int D, int DT> cudaError_t stream_d(const PagedArgs &a, cudaStream_t s) {
    static const cudaError_t attr = cudaFuncSetAttribute(
        stream_kernel<D, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, stream_smem<D>());
    if (attr != cudaSuccess) return attr;
    return launch_paged(stream_kernel<D, DT>, dim3(unsigned(a.prefix_items + a.tail_items)), NW * 32, stream_smem<D>(), s, a);
}

template <int D, int DT> cudaError_t combine_d(const PagedArgs &a, cudaStream_t s) {
    // 16 warps only where a row has many parts
    const int warps = a.n_split + a.n_chunk > 16 ? 16 : 4;
    return launch_paged(combine_kernel<D, DT>, dim3(unsigned(a.n_q_heads), unsigned(a.batch)), 32 * warps, 0, s, a);
}

}  // namespace

cudaError_t launch_paged_stream(int dim, int dtype, const PagedArgs &a, cudaStream_t s) {
    if (a.prefix_items + a.tail_items <= 0) return cudaSuccess;
    KVX_PAGED_DIM(stream_d)
}

cudaError_t launch_paged_combine(int dim, int dtype, const PagedArgs &a, cudaStream_t s) {
    if (a.batch <= 0) return cudaSuccess;
    KVX_PAGED_DIM(combine_d)
}

}  // namespace kvx
