// rms_norm.hip -- the root-mean-square norm of rows with the residual's addition, its gradients, and its 8-bit output.
//
//   h = round(x + residual);  rs = (mean(h^2) + eps)^(-1/2);  y = h rs w        (h = x without a residual)
//   dh_total = rs (w dy - h rs^2 mean(w dy h)) + dh;  dw = sum over rows of dy h rs
//
// Everything is fp32 between the loads and the stores; the norm is taken of the ROUNDED h, which is what the caller gets and what
// the backward pass reads.  Bound by the bytes of the rows: a few operations an element.
#include "odw_common.h"

namespace {

enum { kXBf16 = 1, kHBf16 = 2, kWBf16 = 4 };

__device__ __forceinline__ float ld(const void* p, bool bf, int64_t i) {
    return bf ? __uint_as_float((uint32_t)((const unsigned short*)p)[i] << 16) : ((const float*)p)[i];
}
__device__ __forceinline__ unsigned short f2bf(float f) {      // round to nearest even; NaN stays NaN
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (unsigned short)((u >> 16) | 0x40);
    return (unsigned short)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ float st(void* p, bool bf, int64_t i, float x) {     // returns what was stored
    if (bf) {
        const unsigned short u = f2bf(x);
        ((unsigned short*)p)[i] = u;
        return __uint_as_float((uint32_t)u << 16);
    }
    ((float*)p)[i] = x;
    return x;
}

__device__ __forceinline__ float block_sum(float x, float* part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}
__device__ __forceinline__ uint32_t block_max(uint32_t x, uint32_t* part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)x, off, 64);
        x = x > o ? x : o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    const uint32_t a = part[0] > part[1] ? part[0] : part[1], b = part[2] > part[3] ? part[2] : part[3];
    return a > b ? a : b;
}

// e4m3, rounded to nearest even by the converter; |x| <= 448 or NaN (-> 0x7F).
__device__ __forceinline__ uint8_t to_e4m3(float x) { return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false); }

// A row a workgroup.
template <bool OUT8>
__global__ __launch_bounds__(256) void rms_norm_kernel(const void* x, int64_t ldx, const void* res, int64_t ldr, const void* w, int64_t R,
                                                       int D, float eps, void* y, void* h, float* rstd, float* scale, int types) {
    __shared__ float part[4];
    const bool xb = types & kXBf16, hb = types & kHBf16, wb = types & kWBf16;
    for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < D; i += 256) {
            float v = ld(x, xb, r * ldx + i);
            if (res) v = st(h, hb, r * D + i, v + ld(res, hb, r * ldr + i));
            s += v * v;
        }
        s = block_sum(s, part);
        const float rs = 1.0f / sqrtf(s / (float)D + eps);
        if (rstd && threadIdx.x == 0) rstd[r] = rs;
        uint32_t top = 0;
        for (int i = threadIdx.x; i < D; i += 256) {
            const float v = (res ? ld(h, hb, r * D + i) : ld(x, xb, r * ldx + i)) * rs * (w ? ld(w, wb, i) : 1.0f);
            if (!OUT8) { st(y, xb, r * D + i, v); continue; }
            const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
            top = top > u ? top : u;
        }
        if (OUT8) {
            // the largest word of the magnitudes: a NaN's is above all numbers', so it makes the scale and the whole row NaN
            const float sc0 = __uint_as_float(block_max(top, (uint32_t*)part)) / 448.0f;
            const float sc = sc0 < 1.17549435e-38f ? 1.17549435e-38f : sc0, inv = 1.0f / sc;
            if (threadIdx.x == 0) scale[r] = sc;
            for (int i = threadIdx.x; i < D; i += 256) {
                const float v = (res ? ld(h, hb, r * D + i) : ld(x, xb, r * ldx + i)) * rs * (w ? ld(w, wb, i) : 1.0f);
                ((uint8_t*)y)[r * D + i] = to_e4m3(v * inv);
            }
        }
    }
}

// dx (and dres, when its type is another one); the weight's gradient of this workgroup's rows to part_w (its own row of it).
__global__ __launch_bounds__(256) void rms_norm_bwd_kernel(const void* dy, int64_t ldy, const void* dh, int64_t ldh, const void* h, int64_t ldx,
                                                           const void* w, const float* rstd, int64_t R, int D, void* dx, void* dres,
                                                           float* part_w, int types) {
    __shared__ float part[4];
    const bool xb = types & kXBf16, hb = types & kHBf16, wb = types & kWBf16;
    if (part_w)
        for (int i = threadIdx.x; i < D; i += 256) part_w[(int64_t)blockIdx.x * D + i] = 0.0f;
    for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
        float s = 0.0f;
        const float rs = rstd[r];
        for (int i = threadIdx.x; i < D; i += 256) {
            const float g = ld(dy, xb, r * ldy + i), hv = ld(h, hb, r * ldx + i);
            s += g * (w ? ld(w, wb, i) : 1.0f) * hv;
            if (part_w) part_w[(int64_t)blockIdx.x * D + i] += g * hv * rs;
        }
        s = block_sum(s, part);
        const float k = rs * rs * (s / (float)D);
        for (int i = threadIdx.x; i < D; i += 256) {
            float v = rs * (ld(dy, xb, r * ldy + i) * (w ? ld(w, wb, i) : 1.0f) - ld(h, hb, r * ldx + i) * k);
            if (dh) v += ld(dh, hb, r * ldh + i);
            if (dx) st(dx, xb, r * D + i, v);
            if (dres) st(dres, hb, r * D + i, v);
        }
    }
}

__global__ __launch_bounds__(256) void rms_norm_dw_kernel(const float* part_w, int G, int D, void* dw, int types) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= D) return;
    float s = 0.0f;
    for (int g = 0; g < G; ++g) s += part_w[(int64_t)g * D + i];
    st(dw, types & kWBf16, i, s);
}

constexpr int kBwdGroups = 512;
int bwd_groups(int64_t R) { return (int)(R < kBwdGroups ? R : kBwdGroups); }

int check(const char* what, int64_t R, int D, int types) {
    ODW_REQUIRE(R >= 0 && D >= 1, "%s: bad dims R=%lld D=%d", what, (long long)R, D);
    ODW_REQUIRE(types >= 0 && types < 8, "%s: bad types %d", what, types);
    return ODW_OK;
}

}  // namespace

ODW_EXPORT int odw_rms_norm(const void* x, int64_t ld_x, const void* res, int64_t ld_res, const void* w, int64_t R, int D, float eps, void* y,
                            void* h, float* rstd, int types, void* stream_) {
    const int rc = check("rms_norm", R, D, types);
    if (rc != ODW_OK) return rc;
    if (R == 0) return ODW_OK;
    ODW_REQUIRE(x && y && (!res || h), "rms_norm: null pointer");
    rms_norm_kernel<false><<<(unsigned)(R < 65536 ? R : 65536), 256, 0, (hipStream_t)stream_>>>(x, ld_x, res, ld_res, w, R, D, eps, y, h, rstd,
                                                                                               nullptr, types);
    ODW_CHECK_LAUNCH("rms_norm_kernel");
    return ODW_OK;
}

ODW_EXPORT int odw_rms_norm_fp8(const void* x, int64_t ld_x, const void* res, int64_t ld_res, const void* w, int64_t R, int D, float eps,
                                void* q, float* scale, void* h, int types, void* stream_) {
    const int rc = check("rms_norm_fp8", R, D, types);
    if (rc != ODW_OK) return rc;
    if (R == 0) return ODW_OK;
    ODW_REQUIRE(x && q && scale && (!res || h), "rms_norm_fp8: null pointer");
    rms_norm_kernel<true><<<(unsigned)(R < 65536 ? R : 65536), 256, 0, (hipStream_t)stream_>>>(x, ld_x, res, ld_res, w, R, D, eps, q, h, nullptr,
                                                                                              scale, types);
    ODW_CHECK_LAUNCH("rms_norm_kernel");
    return ODW_OK;
}

ODW_EXPORT int64_t odw_rms_norm_bwd_workspace(int64_t R, int D) { return (int64_t)bwd_groups(R) * D * (int64_t)sizeof(float); }

ODW_EXPORT int odw_rms_norm_bwd(const void* dy, int64_t ld_dy, const void* dh, int64_t ld_dh, const void* h, int64_t ld_h, const void* w,
                                const float* rstd, int64_t R, int D, void* dx, void* dres, void* dw, int types, void* workspace,
                                int64_t workspace_bytes, void* stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const int rc = check("rms_norm_bwd", R, D, types);
    if (rc != ODW_OK) return rc;
    ODW_REQUIRE(R == 0 || (dy && h && rstd), "rms_norm_bwd: null pointer");
    if (dw && workspace_bytes < odw_rms_norm_bwd_workspace(R, D)) {
        odw_set_error("rms_norm_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)odw_rms_norm_bwd_workspace(R, D));
        return ODW_EWORKSPACE;
    }
    ODW_REQUIRE(!dw || R == 0 || workspace, "rms_norm_bwd: null workspace");
    const int G = bwd_groups(R);
    if (R > 0) {
        rms_norm_bwd_kernel<<<G, 256, 0, stream>>>(dy, ld_dy, dh, ld_dh, h, ld_h, w, rstd, R, D, dx, dres, dw ? (float*)workspace : nullptr, types);
        ODW_CHECK_LAUNCH("rms_norm_bwd_kernel");
    }
    if (dw) {
        rms_norm_dw_kernel<<<(D + 255) / 256, 256, 0, stream>>>((const float*)workspace, G, D, dw, types);
        ODW_CHECK_LAUNCH("rms_norm_dw_kernel");
    }
    return ODW_OK;
}
