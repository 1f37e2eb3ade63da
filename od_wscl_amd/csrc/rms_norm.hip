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

// Outputs of the forward pass over this many bytes (the eight L2s together) are stored past the caches (PAST): nothing of them would be
// left there for the next kernel, and the rows coming in keep their place.  Calls one after the other on three sets of rows in turn, us:
// 2000 x 4096 fp32 with residual 23.9 -> 20.0 (6.6 TB/s), 16000 x 4096 bf16 96.1 -> 91.4; forward and backward 201 -> 195.  (A launch by
// itself, as in a trace, is a little slower with it: 24.4 -> 26.0 and 93.5 -> 98.2.  Loads past the caches: slower; stores of the
// backward pass: no difference.)
constexpr int64_t kL2Bytes = (int64_t)32 << 20;

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

// ---- rows that fit the registers ------------------------------------------------------------------------------------------------
// TPR threads hold a row, VPT vectors of V elements each (16 bytes of x's type): one pass over memory, and between load and store the
// row's sum (and largest word) over the lanes -- by cross-lane moves for TPR = 64, through LDS beyond.  Rows of any pitch, width and
// alignment go the same way (the vector loads and stores are declared with their element's alignment, which the memory instructions take
// as well; a row's last, short vector goes by elements): a row's result does not depend on where it lies.  The forms differ in TX (x, y,
// dy, dx) and TH (residual, h, dh, dresidual); the rest is uniform branches.

template <class T, int V> struct Vec {
    typedef T full __attribute__((ext_vector_type(V)));
    typedef full t __attribute__((aligned(sizeof(T))));
};

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(unsigned short x) { return __uint_as_float((uint32_t)x << 16); }
template <class T> __device__ __forceinline__ T down(float x);
template <> __device__ __forceinline__ float down<float>(float x) { return x; }
template <> __device__ __forceinline__ unsigned short down<unsigned short>(float x) { return f2bf(x); }

// `left` elements are there from src on.  fetch() leaves the words as they are (nothing waits for them until they are used).
template <class T, int V>
__device__ __forceinline__ typename Vec<T, V>::full fetch(const T* src, int left) {
    if (left >= V) return *reinterpret_cast<const typename Vec<T, V>::t*>(src);
    typename Vec<T, V>::full u;
#pragma unroll
    for (int j = 0; j < V; ++j) u[j] = j < left ? src[j] : (T)0;
    return u;
}
template <class T, int V>
__device__ __forceinline__ void load(const T* src, int left, float (&x)[V]) {
    const typename Vec<T, V>::full u = fetch<T, V>(src, left);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = up((T)u[j]);
}
template <class T, int V, bool PAST = false>
__device__ __forceinline__ void store(T* dst, int left, const float (&x)[V]) {
    if (left >= V) {
        typename Vec<T, V>::full u;
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = down<T>(x[j]);
        if (PAST) __builtin_nontemporal_store(u, reinterpret_cast<typename Vec<T, V>::t*>(dst));
        else *reinterpret_cast<typename Vec<T, V>::t*>(dst) = u;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < left) dst[j] = down<T>(x[j]);
    }
}
template <int V>
__device__ __forceinline__ void load_w(const void* w, bool bf, int i, int left, float (&x)[V]) {
    if (!w) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = 1.0f;
    } else if (bf) {
        load<unsigned short, V>((const unsigned short*)w + i, left, x);
    } else {
        load<float, V>((const float*)w + i, left, x);
    }
}

// Sum over the threads of a row.  `part` holds a number a wave; the next call but one may use it again (a thread that writes it then has
// passed the barrier of the call between, which every reader of this one has reached).
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) x += part[k];
    }
    return x;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t x, float* part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)x, off, 64);
        x = x > o ? x : o;
    }
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = __uint_as_float(x);
        __syncthreads();
        x = 0;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) {
            const uint32_t o = __float_as_uint(part[k]);
            x = x > o ? x : o;
        }
    }
    return x;
}

// The 8-bit codes are the correctly rounded ones, q = rne(y / (max |y| / 448)), where a quotient rounded to fp32 on the way would go the
// other way round a few times in a million.  The row's factor cancels in it: with t = h w, q = rne(448 t / max |t|).  The fp32 quotient z
// stands for an interval; a thread rounds both its ends, and only rows with a code that is open then go the long way for those codes: t =
// p + e exactly (p the rounded product, e its error by one fma), 448 / max |t| = c + cl in two fp32 numbers, and the product's first 24
// bits in f, the rest in the sign of lo: f with its last bit standing for "and something more" (rounding to odd) rounds to 8 bits as the
// exact product. (Every element the long way: 2000 x 25088 fp32 76 us, for 64.)
__device__ __forceinline__ float times_to_odd(float h, float w, float c, float cl) {
    const float p = h * w, e = fmaf(h, w, -p), z = p * c;
    const float r = fmaf(e, c, fmaf(p, cl, fmaf(p, c, -z)));
    const float f = z + r, lo = r - (f - z);
    uint32_t u = __float_as_uint(f);
    // (c + cl and r are good to 2^-47: nearer to a tie than 2^-44 is a tie)
    if (fabsf(lo) > fabsf(f) * 0x1p-44f) u = (((__float_as_uint(lo) ^ u) >> 31) ? u - 1u : u) | 1u;
    return __uint_as_float(u);
}
__device__ __forceinline__ int codes4(float z0, float z1, float z2, float z3) {
    return __builtin_amdgcn_cvt_pk_fp8_f32(z2, z3, __builtin_amdgcn_cvt_pk_fp8_f32(z0, z1, 0, false), true);
}
__device__ __forceinline__ void store_codes(uint8_t* q, int left, int u) {
    typedef int word __attribute__((aligned(1)));
    if (left >= 4) {
        *reinterpret_cast<word*>(q) = u;
    } else {
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (b < left) q[b] = (uint8_t)(u >> (8 * b));
    }
}

// OUT8: `scale` is given and y are the codes.  (The branch on `scale` is uniform and decided by OUT8; left to run time it keeps what
// belongs to a vector together -- without it the scheduler loads the whole row's weight ahead: 2000 x 25088 bf16 with residual 92
// us for 78, its registers spilt.)
template <class TX, class TH, int TPR, int VPT, int V, bool PAST, bool OUT8>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, TPR > 256 ? 8 : 1)
void rms_norm_row_kernel(const TX* __restrict__ x, int64_t ldx, const TH* __restrict__ res, int64_t ldr, const void* __restrict__ w, int64_t R,
                         int D, float eps, void* __restrict__ y, TH* h, float* __restrict__ rstd, float* __restrict__ scale, int types) {
    constexpr int kRows = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float part[2][TPR > 64 ? TPR / 64 : 1];
    __shared__ int any[TPR > 64 ? TPR / 64 : 1];
    static_assert(TPR == 64 || kRows == 1, "rows that share a workgroup have a wave each");
    const int t = kRows == 1 ? threadIdx.x : threadIdx.x % TPR;
    // (a wave's row is uniform, and the compiler has to know it: scalar row addresses)
    const int64_t r = kRows == 1 ? blockIdx.x : (int64_t)blockIdx.x * kRows + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
    if (r >= R) return;                          // (whole waves; with one row a workgroup never)
    float v[VPT][V];
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int i = (k * TPR + t) * V;
        if (i < D) {
            load<TX, V>(x + r * ldx + i, D - i, v[k]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[k][j] = 0.0f;
        }
    }
    if (res) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int i = (k * TPR + t) * V;
            if (i < D) {
                float a[V];
                load<TH, V>(res + r * ldr + i, D - i, a);
#pragma unroll
                for (int j = 0; j < V; ++j) v[k][j] = up(down<TH>(v[k][j] + a[j]));
                store<TH, V, PAST>(h + r * D + i, D - i, v[k]);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) s += v[k][j] * v[k][j];
    s = row_sum<TPR>(s, part[0]);
    const float rs = 1.0f / sqrtf(s / (float)D + eps);
    if (rstd && t == 0) rstd[r] = rs;
    uint32_t best = 0;                           // (8 bits) the largest word of the products' magnitudes: a NaN's is above all numbers'
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int i = (k * TPR + t) * V;
        if (i < D) {
            float g[V];
            load_w<V>(w, types & kWBf16, i, D - i, g);
            if (!scale) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[k][j] = v[k][j] * rs * g[j];
                store<TX, V, PAST>((TX*)y + r * D + i, D - i, v[k]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[k][j] *= g[j];
                    const uint32_t u = __float_as_uint(v[k][j]) & 0x7FFFFFFFu;
                    best = best > u ? best : u;
                }
            }
        }
    }
    if (!OUT8 || !scale) return;
    const float pm = __uint_as_float(row_max<TPR>(best, part[1]));
    const float sc0 = pm * rs / 448.0f;
    const float sc = sc0 < 1.17549435e-38f ? 1.17549435e-38f : sc0;
    if (t == 0) scale[r] = sc;
    // far off, infinite, NaN (it makes the scale and the whole row NaN) or held up by the smallest scale: by fp32, as it comes
    const bool plain = !(pm > 1e-30f && pm < 1e30f) || sc != sc0;
    const float c = plain ? 1.0f / sc : 448.0f / pm;
    if (plain)
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) v[k][j] *= rs;
    // (z is off by at most 4 * 2^-24 of itself: the product, the largest product, the quotient, their product)
    const float under = plain ? c : c * (1.0f - 0x1p-21f), over = plain ? c : c * (1.0f + 0x1p-21f);
    uint32_t open = 0;                           // fours whose codes are open
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const int i = (k * TPR + t) * V + j;
            if (i >= D) continue;
            const int u = codes4(v[k][j] * under, v[k][j + 1] * under, v[k][j + 2] * under, v[k][j + 3] * under);
            if (u != codes4(v[k][j] * over, v[k][j + 1] * over, v[k][j + 2] * over, v[k][j + 3] * over)) open |= 1u << (k * (V / 4) + j / 4);
            store_codes((uint8_t*)y + r * D + i, D - i, u);
        }
    bool some = __any(open != 0);
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) any[threadIdx.x >> 6] = some;
        __syncthreads();
        some = false;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) some |= any[k] != 0;
    }
    if (!some) return;
    // (the values again, from where they came: their registers hold the products)
    auto value = [&](int i) { return res ? up(h[r * D + i]) : up(x[r * ldx + i]); };
    auto gain = [&](int i) { return w ? ld(w, types & kWBf16, i) : 1.0f; };
    // e of the largest product (of equal ones, in this thread and over the threads, the largest e), as a word that grows with it.  The
    // thread that holds it loads its elements again: looked for in v they would stay in registers until here, and the widest forms spill
    // (2000 x 25088 fp32 69-71 us for 64)
    uint32_t key = 0;
    if (best == __float_as_uint(pm)) {
#pragma clang loop unroll_count(2)
        for (int k = 0; k < VPT; ++k) {
            const int i = (k * TPR + t) * V;
            if (i >= D) break;
            float hv[V], gv[V];
            if (res) load<TH, V>(h + r * D + i, D - i, hv);
            else load<TX, V>(x + r * ldx + i, D - i, hv);
            load_w<V>(w, types & kWBf16, i, D - i, gv);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = hv[j] * gv[j];
                const uint32_t e = __float_as_uint(p < 0.0f ? -fmaf(hv[j], gv[j], -p) : fmaf(hv[j], gv[j], -p));
                const uint32_t word = (e >> 31) ? ~e : e | 0x80000000u;
                if ((__float_as_uint(p) & 0x7FFFFFFFu) == best) key = key > word ? key : word;
            }
        }
    }
    key = row_max<TPR>(key, part[0]);
    const double tmax = (double)pm + (double)__uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
    const double cd = 448.0 / tmax;
    const float ch = (float)cd, cl = (float)(cd - (double)ch);
#pragma clang loop unroll(disable)
    while (open) {
        const int n = __ffs(open) - 1, i = ((n / (V / 4)) * TPR + t) * V + (n % (V / 4)) * 4;
        open &= open - 1;
        float z[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) z[b] = i + b < D ? times_to_odd(value(i + b), gain(i + b), ch, cl) : 0.0f;
        store_codes((uint8_t*)y + r * D + i, D - i, codes4(z[0], z[1], z[2], z[3]));
    }
}

// Rows blockIdx.x, + gridDim.x, ... of a workgroup (TPR = 64: of each of its four waves); the weight's gradient of those rows stays in
// registers and ends in a row of part_w of its own, which rms_norm_dw_kernel sums in order.  While a row's sum goes round, the loads of
// the next row are in flight (kAhead): few groups of rows (little part_w) keep the memory busy.  1024 threads have half the registers
// each: rows over 8 elements a thread are loaded when they are due there, and of the widest ones the weight's gradient lies in LDS (each
// thread its own columns).
constexpr bool wide_row(int tpr, int vpt, int v) { return tpr == 1024 && vpt * v >= 32; }

template <class TX, class TH, int TPR, int VPT, int V>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256)
void rms_norm_bwd_row_kernel(const TX* __restrict__ dy, int64_t ldy, const TH* __restrict__ dh, int64_t ldh, const TH* __restrict__ h,
                             int64_t ldx, const void* __restrict__ w, const float* __restrict__ rstd, int64_t R, int D, TX* __restrict__ dx,
                             TH* __restrict__ dres, float* __restrict__ part_w, int types) {
    constexpr int kRows = TPR > 256 ? 1 : 256 / TPR;
    constexpr bool kWide = wide_row(TPR, VPT, V), kAhead = TPR <= 256 || VPT * V <= 8;
    __shared__ float part[2][TPR > 64 ? TPR / 64 : 1];
    extern __shared__ float acc_lds[];           // kWide: VPT x TPR x V
    typedef typename Vec<float, V>::full Sum;
    const int t = kRows == 1 ? threadIdx.x : threadIdx.x % TPR;
    // (a wave's row is uniform, and the compiler has to know it: scalar row addresses)
    const int own = kRows == 1 ? blockIdx.x : __builtin_amdgcn_readfirstlane(blockIdx.x * kRows + threadIdx.x / TPR);
    const int64_t step = (int64_t)gridDim.x * kRows;
    Sum acc[kWide ? 1 : VPT], wk[kWide ? 1 : VPT];
    Sum* wide_acc = reinterpret_cast<Sum*>(acc_lds);
    typename Vec<TX, V>::full g[VPT], g_next[kAhead ? VPT : 1];
    typename Vec<TH, V>::full v[VPT], v_next[kAhead ? VPT : 1];
    const void* w_now = w;                       // (see the loop)
    auto weight = [&](int k, float (&x)[V]) {
        const int i = (k * TPR + t) * V;
        if (kWide) {
            load_w<V>(w_now, types & kWBf16, i, D - i, x);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = wk[kWide ? 0 : k][j];
        }
    };
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int i = (k * TPR + t) * V;
        if (kWide) {
            wide_acc[k * TPR + t] = (Sum)0.0f;
        } else {
            float x[V];
            load_w<V>(w, types & kWBf16, i, D - i, x);
            acc[kWide ? 0 : k] = (Sum)0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) wk[kWide ? 0 : k][j] = x[j];
        }
        if (kAhead && own < R) {
            g_next[kAhead ? k : 0] = fetch<TX, V>(dy + own * ldy + i, D - i);
            v_next[kAhead ? k : 0] = fetch<TH, V>(h + own * ldx + i, D - i);
        }
    }
    int turn = 0;
    for (int64_t r = own; r < R; r += step, turn ^= 1) {
        const float rs = rstd[r];
        const int64_t next = r + step < R ? r + step : r;
        if (kWide) asm volatile("" : "+s"(w_now));       // loads of w stay in the loop: kept across rows they would not fit the registers
        typename Vec<TH, V>::full d[kAhead ? VPT : 1];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int i = (k * TPR + t) * V;
            if (kAhead) {
                g[k] = g_next[kAhead ? k : 0];
                v[k] = v_next[kAhead ? k : 0];
                if (dh) d[kAhead ? k : 0] = fetch<TH, V>(dh + r * ldh + i, D - i);
                g_next[kAhead ? k : 0] = fetch<TX, V>(dy + next * ldy + i, D - i);
                v_next[kAhead ? k : 0] = fetch<TH, V>(h + next * ldx + i, D - i);
            } else {
                g[k] = fetch<TX, V>(dy + r * ldy + i, D - i);
                v[k] = fetch<TH, V>(h + r * ldx + i, D - i);
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            Sum a = kWide ? wide_acc[k * TPR + t] : acc[kWide ? 0 : k];
            float x[V];
            weight(k, x);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float gj = up((TX)g[k][j]), vj = up((TH)v[k][j]);
                a[j] += gj * vj * rs;
                s += gj * x[j] * vj;
            }
            if (kWide) wide_acc[k * TPR + t] = a;
            else acc[kWide ? 0 : k] = a;
        }
        s = row_sum<TPR>(s, part[turn]);
        const float m = rs * rs * (s / (float)D);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int i = (k * TPR + t) * V;
            if (i >= D) continue;
            if (!kAhead && dh) d[0] = fetch<TH, V>(dh + r * ldh + i, D - i);
            float x[V], a[V];
            weight(k, x);
#pragma unroll
            for (int j = 0; j < V; ++j)
                a[j] = rs * (up((TX)g[k][j]) * x[j] - up((TH)v[k][j]) * m) + (dh ? up((TH)d[kAhead ? k : 0][j]) : 0.0f);
            if (dx) store<TX, V>(dx + r * D + i, D - i, a);
            if (dres) store<TH, V>(dres + r * D + i, D - i, a);
        }
    }
    if (!part_w) return;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int i = (k * TPR + t) * V;
        if (i >= D) continue;
        const Sum a = kWide ? wide_acc[k * TPR + t] : acc[kWide ? 0 : k];
        float x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = a[j];
        store<float, V>(part_w + (int64_t)own * D + i, D - i, x);
    }
}

// 32 columns a workgroup, the rows of part_w over its 32 groups of 32 lanes.
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* __restrict__ part_w, int G, int D, void* __restrict__ dw, int types) {
    constexpr int kCols = 32, kSlices = 1024 / kCols;
    __shared__ float part[kSlices][kCols + 1];
    const int c = threadIdx.x % kCols, slice = threadIdx.x / kCols;
    const int64_t i = (int64_t)blockIdx.x * kCols + c;
    float s = 0.0f;
    if (i < D)
#pragma unroll 8
        for (int g = slice; g < G; g += kSlices) s += part_w[(int64_t)g * D + i];
    part[slice][c] = s;
    __syncthreads();
    // the slices' sums by halves, in one order
    for (int half = kSlices / 2; half > 0; half /= 2) {
        if (slice < half) part[slice][c] += part[slice + half][c];
        __syncthreads();
    }
    if (slice == 0 && i < D) st(dw, types & kWBf16, i, part[0][c]);
}

// ---- rows of any width: the workgroup walks a row as often as it needs it -------------------------------------------------------
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

// ---- which form ------------------------------------------------------------------------------------------------------------------
template <int T_, int K_, int V_> struct Shape { static constexpr int tpr = T_, vpt = K_, v = V_; };
template <class... S> struct Shapes {};

// Rows by width, the first that holds one: a wave a row while a lane needs one or two vectors (no barrier), then 256 and 1024 threads.
// 16000 x 1024 fp32 with a wave and four vectors a lane 49.1 us, with 256 threads 45.7; 4000 x 8192 bf16 with 256 threads and four
// vectors 53.7, with 1024 threads 52.0.  1024 threads of up to 64 registers leave room for a second row on a compute unit: 2000 x 25088
// fp32 to 8 bits 72 us with one row, 56 with two (64 since every code is certain).  The backward pass keeps three numbers an element
// (gradient, h, the weight's gradient) instead of one: fewer elements a thread.
typedef Shapes<Shape<64, 1, 4>, Shape<64, 2, 4>, Shape<256, 1, 4>, Shape<256, 2, 4>, Shape<256, 4, 4>, Shape<256, 8, 4>, Shape<1024, 4, 4>,
               Shape<1024, 5, 4>, Shape<1024, 6, 4>, Shape<1024, 7, 4>, Shape<1024, 8, 4>> Fwd4;
typedef Shapes<Shape<64, 1, 8>, Shape<64, 2, 8>, Shape<256, 1, 8>, Shape<256, 2, 8>, Shape<1024, 1, 8>, Shape<1024, 2, 8>, Shape<1024, 4, 8>> Fwd8;
typedef Shapes<Shape<64, 1, 4>, Shape<64, 2, 4>, Shape<64, 4, 4>, Shape<256, 2, 4>, Shape<256, 4, 4>, Shape<1024, 2, 4>, Shape<1024, 4, 4>,
               Shape<1024, 8, 4>> Bwd4;
typedef Shapes<Shape<64, 1, 8>, Shape<64, 2, 8>, Shape<256, 1, 8>, Shape<256, 2, 8>, Shape<1024, 1, 8>, Shape<1024, 2, 8>, Shape<1024, 4, 8>> Bwd8;

// f(shape) for the first shape that holds D elements; false where none does.
template <class F, class... S>
bool with_shape(int D, Shapes<S...>, F f) {
    return ((D <= S::tpr * S::vpt * S::v ? (f(S()), true) : false) || ...);
}

// Row groups of the backward pass = rows of part_w: enough to fill the chip, few beside the rows.  Measured, us: 16000 x 4096 bf16 (256
// threads a row) 512 groups 101, 768 107, 1024 123; 40000 x 512 bf16 (a wave a row) 1024 groups 66, 2048 45, 4096 49; 3000 x 128 fp32
// 1024 groups 10, 2048 13.
int bwd_groups(int64_t R, int D) {
    if (D <= 1024) return (int)(R < 64 ? R : R < 8192 ? (R + 3) / 4 : 2048);        // (waves)
    const int most = D <= 4096 ? 512 : 256;
    return (int)(R < most ? R : most);
}

int check(const char* what, int64_t R, int D, int types) {
    ODW_REQUIRE(R >= 0 && D >= 1, "%s: bad dims R=%lld D=%d", what, (long long)R, D);
    ODW_REQUIRE(types >= 0 && types < 8, "%s: bad types %d", what, types);
    ODW_REQUIRE(!(types & kHBf16) || (types & kXBf16), "%s: bf16 rows h beside fp32 rows x", what);
    return ODW_OK;
}

template <class TX, class TH>
void forward(const void* x, int64_t ldx, const void* res, int64_t ldr, const void* w, int64_t R, int D, float eps, void* y, void* h, float* rstd,
             float* scale, int types, hipStream_t stream) {
    constexpr int V = sizeof(TX) == 2 ? 8 : 4;
    const bool past = R * D * (int64_t)((scale ? 1 : sizeof(TX)) + (res ? sizeof(TH) : 0)) > kL2Bytes;
    auto launch = [&](auto s) {
        typedef decltype(s) S;
        constexpr int kRows = S::tpr > 256 ? 1 : 256 / S::tpr;
        const auto kernel = scale ? (past ? rms_norm_row_kernel<TX, TH, S::tpr, S::vpt, S::v, true, true>
                                          : rms_norm_row_kernel<TX, TH, S::tpr, S::vpt, S::v, false, true>)
                                  : (past ? rms_norm_row_kernel<TX, TH, S::tpr, S::vpt, S::v, true, false>
                                          : rms_norm_row_kernel<TX, TH, S::tpr, S::vpt, S::v, false, false>);
        // (a launch has fewer than 2^32 threads: rows beyond go to further ones)
        constexpr int64_t kMost = (int64_t)1 << 21;
        for (int64_t r = 0; r < R; r += kMost * kRows) {
            const int64_t n = R - r < kMost * kRows ? R - r : kMost * kRows;
            kernel<<<(unsigned)((n + kRows - 1) / kRows), kRows * S::tpr, 0, stream>>>(
                (const TX*)x + r * ldx, ldx, res ? (const TH*)res + r * ldr : nullptr, ldr, w, n, D, eps,
                (char*)y + r * D * (int64_t)(scale ? 1 : sizeof(TX)), res ? (TH*)h + r * D : nullptr, rstd ? rstd + r : nullptr,
                scale ? scale + r : nullptr, types);
        }
    };
    if constexpr (V == 8) { if (with_shape(D, Fwd8(), launch)) return; }
    else { if (with_shape(D, Fwd4(), launch)) return; }
    const unsigned grid = (unsigned)(R < 65536 ? R : 65536);
    if (scale) rms_norm_kernel<true><<<grid, 256, 0, stream>>>(x, ldx, res, ldr, w, R, D, eps, y, h, rstd, scale, types);
    else rms_norm_kernel<false><<<grid, 256, 0, stream>>>(x, ldx, res, ldr, w, R, D, eps, y, h, rstd, scale, types);
}

// Returns the rows of part_w that were written.
template <class TX, class TH>
int backward(const void* dy, int64_t ldy, const void* dh, int64_t ldh, const void* h, int64_t ldx, const void* w, const float* rstd, int64_t R, int D,
             void* dx, void* dres, float* part_w, int types, hipStream_t stream, hipError_t& status) {
    constexpr int V = sizeof(TX) == 2 ? 8 : 4;
    int groups = bwd_groups(R, D);
    status = hipSuccess;
    auto launch = [&](auto s) {
        typedef decltype(s) S;
        constexpr int kRows = S::tpr > 256 ? 1 : 256 / S::tpr;
        const int grid = groups / kRows > 0 ? groups / kRows : 1;        // (R < kRows: the waves without a row leave zeros)
        groups = grid * kRows;
        const int lds = wide_row(S::tpr, S::vpt, S::v) ? S::tpr * S::vpt * S::v * (int)sizeof(float) : 0;
        const auto kernel = rms_norm_bwd_row_kernel<TX, TH, S::tpr, S::vpt, S::v>;
        if (lds > 0) status = odw_set_max_lds(reinterpret_cast<const void*>(kernel), lds);
        if (status != hipSuccess) return;
        kernel<<<grid, kRows * S::tpr, lds, stream>>>(
            (const TX*)dy, ldy, (const TH*)dh, ldh, (const TH*)h, ldx, w, rstd, R, D, (TX*)dx, (TH*)dres, part_w, types);
    };
    if constexpr (V == 8) { if (with_shape(D, Bwd8(), launch)) return groups; }
    else { if (with_shape(D, Bwd4(), launch)) return groups; }
    rms_norm_bwd_kernel<<<groups, 256, 0, stream>>>(dy, ldy, dh, ldh, h, ldx, w, rstd, R, D, dx, dres, part_w, types);
    return groups;
}

template <class F>
void by_types(int types, F f) {          // f(x's type, h's type)
    if (!(types & kXBf16)) f(float(), float());
    else if (types & kHBf16) f((unsigned short)0, (unsigned short)0);
    else f((unsigned short)0, float());
}

}  // namespace

ODW_EXPORT int odw_rms_norm(const void* x, int64_t ld_x, const void* res, int64_t ld_res, const void* w, int64_t R, int D, float eps, void* y,
                            void* h, float* rstd, int types, void* stream_) {
    const int rc = check("rms_norm", R, D, types);
    if (rc != ODW_OK) return rc;
    if (R == 0) return ODW_OK;
    ODW_REQUIRE(x && y && (!res || h), "rms_norm: null pointer");
    by_types(types, [&](auto tx, auto th) {
        forward<decltype(tx), decltype(th)>(x, ld_x, res, ld_res, w, R, D, eps, y, h, rstd, nullptr, types, (hipStream_t)stream_);
    });
    ODW_CHECK_LAUNCH("rms_norm_kernel");
    return ODW_OK;
}

ODW_EXPORT int odw_rms_norm_fp8(const void* x, int64_t ld_x, const void* res, int64_t ld_res, const void* w, int64_t R, int D, float eps,
                                void* q, float* scale, void* h, int types, void* stream_) {
    const int rc = check("rms_norm_fp8", R, D, types);
    if (rc != ODW_OK) return rc;
    if (R == 0) return ODW_OK;
    ODW_REQUIRE(x && q && scale && (!res || h), "rms_norm_fp8: null pointer");
    by_types(types, [&](auto tx, auto th) {
        forward<decltype(tx), decltype(th)>(x, ld_x, res, ld_res, w, R, D, eps, q, h, nullptr, scale, types, (hipStream_t)stream_);
    });
    ODW_CHECK_LAUNCH("rms_norm_kernel");
    return ODW_OK;
}

// (+ 3: a workgroup of four rows writes four rows of part_w)
ODW_EXPORT int64_t odw_rms_norm_bwd_workspace(int64_t R, int D) {
    return R > 0 ? (int64_t)(bwd_groups(R, D) + 3) * D * (int64_t)sizeof(float) : 0;
}

ODW_EXPORT int odw_rms_norm_bwd(const void* dy, int64_t ld_dy, const void* dh, int64_t ld_dh, const void* h, int64_t ld_h, const void* w,
                                const float* rstd, int64_t R, int D, void* dx, void* dres, void* dw, int types, void* workspace,
                                int64_t workspace_bytes, void* stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const int rc = check("rms_norm_bwd", R, D, types);
    if (rc != ODW_OK) return rc;
    ODW_REQUIRE(R == 0 || (dy && h && rstd), "rms_norm_bwd: null pointer");
    if (dw && R > 0 && workspace_bytes < odw_rms_norm_bwd_workspace(R, D)) {
        odw_set_error("rms_norm_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)odw_rms_norm_bwd_workspace(R, D));
        return ODW_EWORKSPACE;
    }
    ODW_REQUIRE(!dw || R == 0 || workspace, "rms_norm_bwd: null workspace");
    int groups = 0;
    hipError_t status = hipSuccess;
    if (R > 0) {
        by_types(types, [&](auto tx, auto th) {
            groups = backward<decltype(tx), decltype(th)>(dy, ld_dy, dh, ld_dh, h, ld_h, w, rstd, R, D, dx, dres, dw ? (float*)workspace : nullptr,
                                                          types, stream, status);
        });
        ODW_CHECK_HIP(status, "rms_norm_bwd attr");
        ODW_CHECK_LAUNCH("rms_norm_bwd_kernel");
    }
    if (dw) {
        rms_norm_dw_kernel<<<(unsigned)(((int64_t)D + 31) / 32), 1024, 0, stream>>>((const float*)workspace, groups, D, dw, types);
        ODW_CHECK_LAUNCH("rms_norm_dw_kernel");
    }
    return ODW_OK;
}
