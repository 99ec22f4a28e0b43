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

// Cosines and sines of pairs [8 c, 8 c + 8) of a token.
__device__ __forceinline__ bool load_angles(const RotArgs &a, int token, int c, float (&co)[8], float (&si)[8]) {
    const int half = a.rot_dim >> 1;
    uint2 ax = make_uint2(0u, 0u);
    if (a.axis != nullptr) ax = __ldg(reinterpret_cast<const uint2 *>(a.axis + 8 * c));
    const uint32_t first = ax.x & 0xFFu;
    if (ax.x == first * 0x01010101u && ax.y == ax.x) {  // the eight pairs turn about one axis
        const int p = table_row(a, token, int(first));
        if (p < 0) return false;
        const float4 *pc = reinterpret_cast<const float4 *>(a.cos + int64_t(p) * half + 8 * c);
        const float4 *ps = reinterpret_cast<const float4 *>(a.sin + int64_t(p) * half + 8 * c);
        const float4 c0 = __ldg(pc), c1 = __ldg(pc + 1), s0 = __ldg(ps), s1 = __ldg(ps + 1);
        co[0] = c0.x, co[1] = c0.y, co[2] = c0.z, co[3] = c0.w, co[4] = c1.x, co[5] = c1.y, co[6] = c1.z, co[7] = c1.w;
        si[0] = s0.x, si[1] = s0.y, si[2] = s0.z, si[3] = s0.w, si[4] = s1.x, si[5] = s1.y, si[6] = s1.z, si[7] = s1.w;
        return true;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int p = table_row(a, token, int(((i < 4 ? ax.x : ax.y) >> (8 * (i & 3))) & 0xFFu));
        if (p < 0) return false;
        co[i] = __ldg(a.cos + int64_t(p) * half + 8 * c + i);
        si[i] = __ldg(a.sin + int64_t(p) * half + 8 * c + i);
    }
    return true;
}

// (a, b) -> (a cos - b sin, b cos + a sin), each product and sum rounded in FP32.
__device__ __forceinline__ void turn(float &x, float &y, float c, float s) {
    const float u = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
    x = u;
}

// One thread per (token, head, 16 values): eight pairs -- two 16-byte pieces rot_dim / 2 apart, or
// adjacent when interleaved -- or 16 values copied.  The operator moves four bytes a value and
// computes three operations, so it is bound by HBM (and by the launch for a few tokens); the
// tables' rows are shared by all heads of a token, which are neighbours in a CTA, and come from L1.
template <int DT>
__global__ void __launch_bounds__(256) rotate_vec_kernel(const RotArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int nc = a.dim >> 4, per = a.heads * nc;
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
        const bool rot = sg.rotated && 16 * c < a.rot_dim;
        int o0 = 16 * c, o1 = 16 * c + 8;
        if (rot && !a.interleaved) o0 = 8 * c, o1 = 8 * c + (a.rot_dim >> 1);
        uint4 x = *reinterpret_cast<const uint4 *>(in + o0);
        uint4 y = *reinterpret_cast<const uint4 *>(in + o1);
        if (rot) {
            float co[8], si[8];
            if (!load_angles(a, token, c, co, si)) continue;
            uint32_t *xw = &x.x, *yw = &y.x;
            const float sign = a.inverse ? -1.f : 1.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 u = Half2<DT>::up(xw[j]), w = Half2<DT>::up(yw[j]);
                if (a.interleaved) {
                    turn(u.x, u.y, co[j], sign * si[j]);
                    turn(w.x, w.y, co[4 + j], sign * si[4 + j]);
                } else {
                    turn(u.x, w.x, co[2 * j], sign * si[2 * j]);
                    turn(u.y, w.y, co[2 * j + 1], sign * si[2 * j + 1]);
                }
                xw[j] = Half2<DT>::down(u.x, u.y);
                yw[j] = Half2<DT>::down(w.x, w.y);
            }
        }
        *reinterpret_cast<uint4 *>(out + o0) = x;
        *reinterpret_cast<uint4 *>(out + o1) = y;
    }
}

// The same for any even width, stride and alignment: one thread per (token, head, pair of values).
template <int DT>
__global__ void __launch_bounds__(256) rotate_any_kernel(const RotArgs a) {
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

cudaError_t launch_rotate(int dtype, bool vec, const RotArgs &args, cudaStream_t s) {
    if (args.n_tokens <= 0 || args.heads <= 0) return cudaSuccess;
    RotArgs a = args;
    const int per = a.heads * (vec ? a.dim >> 4 : a.dim >> 1);
    a.tokens_per_cta = per >= 256 ? 1 : 256 / per;
    // programmatic dependent launch: the kernel waits for the grid before it
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned((a.n_tokens + a.tokens_per_cta - 1) / a.tokens_per_cta));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (dtype == KVX_DTYPE_BF16)
        return cudaLaunchKernelEx(&cfg, vec ? rotate_vec_kernel<KVX_DTYPE_BF16> : rotate_any_kernel<KVX_DTYPE_BF16>, a);
    return cudaLaunchKernelEx(&cfg, vec ? rotate_vec_kernel<KVX_DTYPE_FP16> : rotate_any_kernel<KVX_DTYPE_FP16>, a);
}

}  // namespace kvx
