// rotate.cu -- position rotation of query and key heads, alone or on the way into a paged cache.
#include "paged.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace kvx {
namespace {

template <int DT> struct Half2;
template <> struct Half2<KVX_DTYPE_BF16> {
    static __device__ __forceinline__ float2 up(uint32_t x) {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <> struct Half2<KVX_DTYPE_FP16> {
    static __device__ __forceinline__ float2 up(uint32_t x) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&x));
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <int DT> __device__ __forceinline__ float up1(uint16_t x) { return Half2<DT>::up(x).x; }
template <int DT> __device__ __forceinline__ uint16_t down1(float a) { return uint16_t(Half2<DT>::down(a, 0.f)); }

// Where a head of one token goes.  false: a padding token's K or V (negative slot), or a slot
// outside the pools (reported).
__device__ __forceinline__ bool dest(const RotArgs &a, const RotSeg &sg, int token, int head, uint16_t *&out) {
    if (sg.pool == 0) {
        out = sg.dst + int64_t(token) * sg.dst_token + int64_t(head) * sg.dst_head;
        return true;
    }
    const int64_t slot = __ldg(a.slots + token);
    if (slot < 0) return false;
    int64_t page;
    int32_t place;
    a.pool.split.at(slot, page, place);
    if (page >= a.pool.n_pages) {
        report(a.status, KVX_ERR_RUNTIME, DERR_SLOT);
        return false;
    }
    out = (sg.pool == 1 ? a.pool.k : a.pool.v) + page * a.pool.page_stride + int64_t(place) * a.pool.token_stride +
          int64_t(head) * a.pool.head_stride;
    return true;
}

// Row of the tables for pair i of a token, or -1 (reported).
__device__ __forceinline__ int table_row(const RotArgs &a, int token, int axis) {
    const int p = axis < a.n_axes ? __ldg(a.pos + int64_t(axis) * a.pos_stride + token) : -1;
    if (unsigned(p) < unsigned(a.n_pos)) return p;
    report(a.status, KVX_ERR_RUNTIME, DERR_POSITION);
    return -1;
}

// Cosines and sines of pairs p .. p + 3 of a token (p a multiple of 4).
__device__ __forceinline__ bool load_angles(const RotArgs &a, int token, int p, float *co, float *si) {
    const int half = a.rot_dim >> 1;
    const uint32_t ax = a.axis != nullptr ? __ldg(reinterpret_cast<const uint32_t *>(a.axis + p)) : 0u;
    const uint32_t first = ax & 0xFFu;
    if (ax == first * 0x01010101u) {  // the four pairs turn about one axis
        const int row = table_row(a, token, int(first));
        if (row < 0) return false;
        const float4 c = __ldg(reinterpret_cast<const float4 *>(a.cos + int64_t(row) * half + p));
        const float4 s = __ldg(reinterpret_cast<const float4 *>(a.sin + int64_t(row) * half + p));
        co[0] = c.x, co[1] = c.y, co[2] = c.z, co[3] = c.w;
        si[0] = s.x, si[1] = s.y, si[2] = s.z, si[3] = s.w;
        return true;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = table_row(a, token, int((ax >> (8 * i)) & 0xFFu));
        if (row < 0) return false;
        co[i] = __ldg(a.cos + int64_t(row) * half + p + i);
        si[i] = __ldg(a.sin + int64_t(row) * half + p + i);
    }
    return true;
}

// (a, b) -> (a cos - b sin, b cos + a sin), each product and sum rounded in FP32.
__device__ __forceinline__ void turn(float &x, float &y, float c, float s) {
    const float u = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
    x = u;
}

// 16 bytes that are read or written once: past L1, which the tables' rows are to stay in.
__device__ __forceinline__ uint4 load_once(const uint16_t *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void store_once(uint16_t *p, const uint4 &v) {
    asm volatile("st.global.L1::no_allocate.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Eight pairs of a head, their two pieces in x and y: pairs (x[i], y[i]), or the adjacent values of x
// and then of y.
template <int DT, bool INTER>
__device__ __forceinline__ void turn8(uint4 &x, uint4 &y, const float (&co)[8], const float (&si)[8]) {
    uint32_t *xw = &x.x, *yw = &y.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float2 u = Half2<DT>::up(xw[j]), w = Half2<DT>::up(yw[j]);
        if constexpr (INTER) {
            turn(u.x, u.y, co[j], si[j]);
            turn(w.x, w.y, co[4 + j], si[4 + j]);
        } else {
            turn(u.x, w.x, co[2 * j], si[2 * j]);
            turn(u.y, w.y, co[2 * j + 1], si[2 * j + 1]);
        }
        xw[j] = Half2<DT>::down(u.x, u.y);
        yw[j] = Half2<DT>::down(w.x, w.y);
    }
}

// Where a thread's two pieces of a head are (elements): half the rotated part apart, or half the rest,
// or half of a head that is copied whole, so that a warp's accesses are whole lines either way.
struct Pieces {
    int first, apart;
    bool turned;
};
__device__ __forceinline__ Pieces pieces_of(const RotArgs &a, const RotSeg &sg, int c) {
    const int nr = sg.rotated ? a.rot_dim >> 4 : 0;  // pieces of the rotated part come first
    if (c < nr) return {8 * c, a.rot_dim >> 1, true};
    return {16 * nr + 8 * (c - nr), (a.dim - 16 * nr) >> 1, false};
}
template <bool INTER> __device__ __forceinline__ bool load_angles8(const RotArgs &a, int token, int c, float (&co)[8], float (&si)[8]) {
    const bool ok = INTER ? load_angles(a, token, 4 * c, co, si) && load_angles(a, token, (a.rot_dim >> 2) + 4 * c, co + 4, si + 4)
                          : load_angles(a, token, 8 * c, co, si) && load_angles(a, token, 8 * c + 4, co + 4, si + 4);
    if (a.inverse) {
#pragma unroll
        for (int j = 0; j < 8; ++j) si[j] = -si[j];
    }
    return ok;
}

// Many tokens.  One thread per (token, 16 values of a head, head slot): it turns or copies them in
// every head_slots-th head.  The operator moves four bytes a value and computes three operations: HBM
// bounds it as long as a head's piece costs few instructions, so the angles are loaded and every
// division is done once a thread.  On one B200: 16384 tokens of 32 + 2 x 8 heads of 128 into pages
// 65.5 us (6.15 TB/s), 32768 tokens of 32 heads of 128 84 us (6.4 TB/s); with one thread a head and
// piece 115 and 152 us, with four heads a thread instead of eight 67.5 and 85.
template <int DT, bool INTER>
__global__ void __launch_bounds__(256, 4) rotate_many_kernel(const __grid_constant__ RotArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int G = 2;  // heads whose loads are in flight together
    const int nc = a.dim >> 4;
    const int c = int(threadIdx.x) % nc, r = int(threadIdx.x) / nc;
    const int slot = r % a.head_slots, token = int(blockIdx.x) * a.tokens_per_cta + r / a.head_slots;
    if (r >= a.tokens_per_cta * a.head_slots || token >= a.n_tokens) return;
    float co[8], si[8];
    // (a padding token without queries turns nothing, and its position is not looked at)
    const bool turns = a.seg[0].pool == 0 || __ldg(a.slots + token) >= 0;
    const bool angles = 16 * c >= a.rot_dim || (turns && load_angles8<INTER>(a, token, c, co, si));
#pragma unroll
    for (int g = 0; g < 3; ++g) {
        const RotSeg &sg = a.seg[g];
        const Pieces p = pieces_of(a, sg, c);
        uint16_t *out;
        if (slot >= sg.heads || (p.turned && !angles) || !dest(a, sg, token, slot, out)) continue;
        const uint16_t *in = sg.src + int64_t(token) * sg.src_token + int64_t(slot) * sg.src_head + p.first;
        out += p.first;
        const int64_t in_step = int64_t(a.head_slots) * sg.src_head,
                      out_step = int64_t(a.head_slots) * (sg.pool != 0 ? a.pool.head_stride : sg.dst_head);
        for (int h = slot; h < sg.heads; h += G * a.head_slots) {
            uint4 x[G], y[G];
#pragma unroll
            for (int k = 0; k < G; ++k)
                if (h + k * a.head_slots < sg.heads) x[k] = load_once(in + k * in_step), y[k] = load_once(in + k * in_step + p.apart);
#pragma unroll
            for (int k = 0; k < G; ++k)
                if (h + k * a.head_slots < sg.heads) {
                    if (p.turned) turn8<DT, INTER>(x[k], y[k], co, si);
                    store_once(out + k * out_step, x[k]);
                    store_once(out + k * out_step + p.apart, y[k]);
                }
            in += G * in_step;
            out += G * out_step;
        }
    }
}

// Few tokens: one thread per (token, head of any kind, 16 values), so that nothing follows anything but
// the chain position -> angles.  One token of 14 + 2 x 2 heads of 64: 2 us, the launch.
template <int DT, bool INTER>
__global__ void __launch_bounds__(256) rotate_few_kernel(const __grid_constant__ RotArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const unsigned nc = unsigned(a.dim) >> 4, i = blockIdx.x * 256u + threadIdx.x, r = i / nc;
    const int c = int(i - r * nc), token = int(r / unsigned(a.heads));
    if (token >= a.n_tokens) return;
    int head = int(r) - token * a.heads, g = 0;
    if (head >= a.seg[0].heads) {
        head -= a.seg[0].heads, g = 1;
        if (head >= a.seg[1].heads) head -= a.seg[1].heads, g = 2;
    }
    const RotSeg &sg = a.seg[g];
    const Pieces p = pieces_of(a, sg, c);
    const uint16_t *in = sg.src + int64_t(token) * sg.src_token + int64_t(head) * sg.src_head + p.first;
    uint4 x = load_once(in), y = load_once(in + p.apart);
    uint16_t *out;
    if (!dest(a, sg, token, head, out)) return;
    if (p.turned) {
        float co[8], si[8];
        if (!load_angles8<INTER>(a, token, c, co, si)) return;
        turn8<DT, INTER>(x, y, co, si);
    }
    store_once(out + p.first, x);
    store_once(out + p.first + p.apart, y);
}

// The same for any even width, stride and alignment: one thread per (token, head, pair of values), two
// bytes an access.  32768 tokens of 32 heads of 128, 72 of them rotated: 418 us (1.3 TB/s), where 64 rotated
// take 84 in the kernel above; 20000 of 9 heads of 32 with 24 rotated: 25 us.
template <int DT>
__global__ void __launch_bounds__(256) rotate_any_kernel(const __grid_constant__ RotArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int nc = a.dim >> 1, per = a.heads * nc, half = a.rot_dim >> 1;
    const int t0 = blockIdx.x * a.tokens_per_cta;
    const int n = min(a.tokens_per_cta, a.n_tokens - t0) * per;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int token = t0 + i / per;
        int r = i % per;
        int head = r / nc, sgi = 0;
        const int c = r - head * nc;
        if (head >= a.seg[0].heads) {
            head -= a.seg[0].heads;
            sgi = 1;
            if (head >= a.seg[1].heads) head -= a.seg[1].heads, sgi = 2;
        }
        const RotSeg &sg = a.seg[sgi];
        uint16_t *out;
        if (!dest(a, sg, token, head, out)) continue;
        const uint16_t *in = sg.src + int64_t(token) * sg.src_token + int64_t(head) * sg.src_head;
        const bool rot = sg.rotated && c < half;
        const int o0 = rot && !a.interleaved ? c : 2 * c, o1 = rot && !a.interleaved ? c + half : 2 * c + 1;
        uint16_t x = in[o0], y = in[o1];
        if (rot) {
            const int p = table_row(a, token, a.axis != nullptr ? int(__ldg(a.axis + c)) : 0);
            if (p < 0) continue;
            float u = up1<DT>(x), w = up1<DT>(y);
            const float s = __ldg(a.sin + int64_t(p) * half + c);
            turn(u, w, __ldg(a.cos + int64_t(p) * half + c), a.inverse ? -s : s);
            x = down1<DT>(u);
            y = down1<DT>(w);
        }
        out[o0] = x;
        out[o1] = y;
    }
}

}  // namespace

namespace {
template <int DT> void (*kernel_of(const RotArgs &a, bool vec, bool many))(const RotArgs) {
    if (!vec) return rotate_any_kernel<DT>;
    if (many) return a.interleaved ? rotate_many_kernel<DT, true> : rotate_many_kernel<DT, false>;
    return a.interleaved ? rotate_few_kernel<DT, true> : rotate_few_kernel<DT, false>;
}
}  // namespace

cudaError_t launch_rotate(int dtype, bool vec, const RotArgs &args, cudaStream_t s) {
    if (args.n_tokens <= 0 || args.heads <= 0) return cudaSuccess;
    RotArgs a = args;
    const int nc = a.dim >> 4;
    // a thread for every piece while they fill the device only a few times over
    const int64_t pieces = int64_t(a.n_tokens) * a.heads * nc;
    const bool many = vec && pieces > int64_t(1) << 20;
    int64_t ctas = (pieces + 255) / 256;
    if (many || !vec) {
        const int slots = vec ? 256 / nc : 0, per = a.heads * (a.dim >> 1);
        if (many) {
            int most = 0;
            for (const RotSeg &sg : a.seg) most = sg.heads > most ? sg.heads : most;
            a.head_slots = (most + 7) / 8 < slots ? (most + 7) / 8 : slots;
            a.tokens_per_cta = slots / a.head_slots;
        } else {
            a.tokens_per_cta = per >= 256 ? 1 : 256 / per;
        }
        ctas = (a.n_tokens + a.tokens_per_cta - 1) / a.tokens_per_cta;
    }
    // programmatic dependent launch: the kernel waits for the grid before it
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, dtype == KVX_DTYPE_BF16 ? kernel_of<KVX_DTYPE_BF16>(a, vec, many) : kernel_of<KVX_DTYPE_FP16>(a, vec, many), a);
}

}  // namespace kvx
