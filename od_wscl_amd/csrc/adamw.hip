// adamw.hip -- the AdamW update of many tensors in one launch (states in fp32, or in 8-bit floats with block scales), and the
// global gradient norm it is clipped by.
//
// A launch takes up to kMaxTensors tensors (the norm kNormTensors): their pointers and sizes travel in the kernel's arguments (no table
// in device memory to upload, nothing to keep alive for a captured launch).  The tensors are cut into chunks; a workgroup finds the
// tensor of its chunk with one load of the chunks' prefix, a lane a tensor (the arguments lie in host memory: a bisection's six dependent
// loads of them were half the time of a small launch).
//
// Both are bound by the bytes: an element's update is ~20 operations on 28 bytes with fp32 states (30 with a bf16 copy of p), ~70 on 16
// (18) with 8-bit ones.  153 M parameters in 42 tensors with copies: 796 us (5.8 TB/s) and 463 us (5.9 TB/s); their gradients' norm
// 88 us (7.0 TB/s), their scaling 220 us (5.5 TB/s).  A launch of a million elements in 48 small tensors takes 8-10 us.
#include "odw_common.h"
#include "odw_rng.h"
#include <math.h>

namespace {

constexpr int kMaxTensors = 48, kNormTensors = 160;      // (the arguments stay under 4 KB)
constexpr int kBlock = 256;              // elements that share a scale: one wave, four elements a lane
// A workgroup's four waves have a whole chunk's loads in flight: 4 blocks a wave of fp32 states, 2 of 8-bit ones (more registers a
// block).  153 M parameters with bf16 copies, us: fp32 states 825 (2 blocks), 796 (4), 819 (8); 8-bit states 493 (1), 468 (2), 475 (4);
// chunks of several rounds are slower (4096 elements by 2 blocks: 485; 16384: 528), and so are plain loads (522) or plain stores (511)
// for the nontemporal ones.
constexpr int unroll(bool bits8) { return bits8 ? 2 : 4; }
constexpr int chunk_of(bool bits8) { return unroll(bits8) * 4 * kBlock; }
constexpr int kMaxGrid = 1 << 23;        // (a launch has fewer than 2^32 threads; the update's workgroups walk on)
constexpr int kNormChunk = 16384;        // the same of the norm: fewer partial sums for the workgroup that adds them
constexpr int kThreads = 256;

enum { kPBf16 = 1, kGBf16 = 2, kVToZero = 4 };

struct Tensor {
    void* p;
    const void* g;
    void* m;
    void* v;
    uint8_t* e;                          // exponents + 127 of the block scales, (m, v) pairs
    unsigned short* copy;                // bf16 copy of p, or null
    int64_t n;
    uint64_t first;                      // the random counter of element 0
    float lr, wd;
    int flags;
};

struct Args {
    Tensor t[kMaxTensors];
    int chunk0[kMaxTensors];             // chunks of the tensors before each
    int count, chunks;
    float b1, b2, omb1, omb2, eps, c1, c2, mult;
    uint32_t k0, k1;
    const float* scale;                  // device factor of the gradients, or null
    const float* bias;                   // device bias corrections and step (odw_adamw_advance), or null: c1, c2
};

struct NormArgs {
    const void* g[kNormTensors];
    int64_t n[kNormTensors];
    int chunk0[kNormTensors];
    uint8_t flags[kNormTensors];
    int count, chunks;
};
static_assert(sizeof(Args) <= 4096 && sizeof(NormArgs) <= 4096 - 64, "kernel arguments");

__device__ __forceinline__ float bf2f(unsigned short h) { return __uint_as_float((uint32_t)h << 16); }
__device__ __forceinline__ unsigned short f2bf(float f) {      // round to nearest even; NaN stays NaN
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (unsigned short)((u >> 16) | 0x40);
    return (unsigned short)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// The tensor that a chunk lies in, the last one whose first chunk is not behind it: lane l looks at tensors l, l + 64, ...
template <int N>
struct Prefix {
    int first[(N + 63) / 64];
    __device__ __forceinline__ Prefix(const int* chunk0, int count) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < (N + 63) / 64; ++k) first[k] = lane + 64 * k < count ? chunk0[lane + 64 * k] : INT32_MAX;
    }
    __device__ __forceinline__ int tensor_of(int c) const {
        int n = 0;
#pragma unroll
        for (int k = 0; k < (N + 63) / 64; ++k) n += __popcll(__ballot(first[k] <= c));
        return n - 1;
    }
    __device__ __forceinline__ int chunk0_of(int t) const {
        int x = __builtin_amdgcn_readlane(first[0], t & 63);
#pragma unroll
        for (int k = 1; k < (N + 63) / 64; ++k) x = t >= 64 * k ? __builtin_amdgcn_readlane(first[k], t & 63) : x;
        return x;
    }
};

// A wave's 256 elements, four consecutive ones a lane, by vectors declared with their element's alignment, which the memory instructions
// take as well: tensors may start at any element.  Nothing is read twice: all loads and stores are marked nontemporal.
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned short us4 __attribute__((ext_vector_type(4)));
typedef f4 f4_any __attribute__((aligned(4)));
typedef us4 us4_any __attribute__((aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// `left` = elements from src on (FULL: at least 256 -- nothing to check; else it is the same for the whole wave, and may be negative).
template <bool BF, bool FULL>
struct Four {
    union { f4 f; us4 h; } u;
    __device__ __forceinline__ void load(const void* src, int lane, int left) {
        if (FULL || left >= kBlock) {
            if (BF) u.h = __builtin_nontemporal_load((const us4_any*)src + lane);
            else u.f = __builtin_nontemporal_load((const f4_any*)src + lane);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * lane + j;
                if (BF) u.h[j] = i < left ? ((const unsigned short*)src)[i] : (unsigned short)0;
                else u.f[j] = i < left ? ((const float*)src)[i] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ float get(int j) const { return BF ? bf2f(u.h[j]) : u.f[j]; }
    __device__ __forceinline__ void set(int j, float x) { if (BF) u.h[j] = f2bf(x); else u.f[j] = x; }
    __device__ __forceinline__ void store(void* dst, int lane, int left) const {
        if (FULL || left >= kBlock) {
            if (BF) __builtin_nontemporal_store(u.h, (us4_any*)dst + lane);
            else __builtin_nontemporal_store(u.f, (f4_any*)dst + lane);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * lane + j;
                if (i >= left) continue;
                if (BF) ((unsigned short*)dst)[i] = u.h[j];
                else ((float*)dst)[i] = u.f[j];
            }
        }
    }
};

template <bool FULL>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* src, int lane, int left) {
    if (FULL || left >= kBlock) return __builtin_nontemporal_load((const u32_any*)src + lane);
    uint32_t u = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (4 * lane + j < left) u |= (uint32_t)src[4 * lane + j] << (8 * j);
    return u;
}

template <bool FULL>
__device__ __forceinline__ void store_codes(uint8_t* dst, int lane, int left, uint32_t u) {
    if (FULL || left >= kBlock) {
        __builtin_nontemporal_store(u, (u32_any*)dst + lane);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (4 * lane + j < left) dst[4 * lane + j] = (uint8_t)(u >> (8 * j));
}

// ---- the 8-bit states ---------------------------------------------------------------------------------------------------------
// m: sign, 4 exponent bits (bias 7), 3 mantissa bits, largest value 1.75 * 2^8, no infinity, 0x7F = NaN.
// v: sign, 5 exponent bits (bias 15), 2 mantissa bits, largest value 1.75 * 2^15, 0x7F = NaN (0x7C = infinity is not written).
// Value = code * 2^(e - 127).  Decay moves v by 0.1 % a step and the formats' steps are 12-25 %: rounded to nearest, v would stay
// where it is; the codes are rounded stochastically, so that their expectation moves.  The scales are powers of two: then the grid
// is the same from step to step, a stored value lies on it, and the rounding's variance a step is (relative change) x (grid
// step) instead of (grid step)^2 / 6 -- summed over v's memory of 1 / (1 - beta2) steps a standard deviation of ~0.15 of sqrt(v), without
// a bias of v, instead of one larger than v itself.
// A v that is not zero is held as 2^-16 of its scale at least.  An element whose gradients are far below its block's largest can have
// its m rounded up to the smallest number, at most 2^-16.8 of the block's largest m; over a v held as zero that would be an update of any
// size -- over 2^-31.8 of the block's largest v, whose root is 2^-15.9 of the largest root, it is at most 4 lr: the largest m is at most
// (1 - b1) / sqrt((1 - b2) (1 - b1^2 / b2)) = 7.3 largest roots for beta = 0.9, 0.999 (Cauchy and Schwarz on the two sums of past
// gradients).  (kVToZero: v is rounded to zero like any other value, without that bound.)
// All of it is integer arithmetic on the fp32 words: the same bits whatever the launch geometry.
template <int BIAS, int MANT>
__device__ __forceinline__ uint32_t encode8(float x, float inv_scale, uint32_t rand16, uint32_t least, bool any_bad) {
    constexpr int kDrop = 23 - MANT;
    const float y = fabsf(x) * inv_scale;
    const uint32_t u = __float_as_uint(y);
    // the value in units of 2^-kDrop grid steps: the fp32 word, rebiased, or below the smallest normal number fixed point (cut: the
    // comparison with the random number is the exact one)
    const uint32_t word = u < ((uint32_t)(128 - BIAS) << 23) ? (uint32_t)(y * __uint_as_float((uint32_t)(149 + BIAS) << 23))
                                                             : u - ((uint32_t)(127 - BIAS) << 23);
    uint32_t code = (word + (rand16 << (kDrop - 16)) + (1u << (kDrop - 17))) >> kDrop;
    if (code < least && x != 0.0f) code = least;
    if (any_bad && (__float_as_uint(x) & 0x7F800000u) == 0x7F800000u) code = 0x7Fu;
    return code | ((__float_as_uint(x) >> 31) << 7);
}

// The scale of 256 values whose largest finite magnitude has the word `mx`: 2^(exponent - TOP), twice that where the mantissa is
// over 1.75, which the format's largest value 1.75 * 2^TOP could not hold.
template <int TOP>
__device__ __forceinline__ int block_exponent(uint32_t mx) {
    int e = (int)(mx >> 23) - TOP + ((mx & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1 : e;
}

// Largest of a wave's words, as a scalar: shifts within the rows of 16 lanes, then the rows' last lanes broadcast onwards.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#define ODW_MAX_STEP(CTRL)                                                                              \
    {                                                                                                   \
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);      \
        x = x > o ? x : o;                                                                              \
    }
    ODW_MAX_STEP(0x111) ODW_MAX_STEP(0x112) ODW_MAX_STEP(0x114) ODW_MAX_STEP(0x118)      // row_shr 1, 2, 4, 8
    ODW_MAX_STEP(0x142) ODW_MAX_STEP(0x143)                                              // row_bcast 15, 31
#undef ODW_MAX_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

struct Step { float gs, rc2, step, decay; uint32_t k1, least_v; };

// p, g, m, v in, p, m, v (and p's bf16 copy) out, for U blocks of 256 elements `stride` apart, `left0` elements being there from the
// first one's start: all loads first.  The averages are formed with one rounding an operation (no contraction), in the order m b1 + g (1
// - b1), v b2 + g g (1 - b2); the ratio with the hardware's root and reciprocal (1 ulp each: 2^-22 of a step of lr is far below p's
// rounding; eps keeps the reciprocal's argument above 1e-15 and makes roots of subnormal numbers, which the instruction takes for zero,
// irrelevant).
template <bool BITS8, bool PBF, bool GBF, bool FULL, int U>
__device__ __forceinline__ void update(const Args& a, const Tensor& t, const Step& s, int64_t base, int stride, int lane, int left0) {
    Four<PBF, FULL> p[U];
    Four<GBF, FULL> g[U];
    Four<false, FULL> fm[U], fv[U];
    uint32_t qm[U], qv[U], ee[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t o = base + u * stride;
        const int left = left0 - u * stride;
        if (!FULL && left <= 0) continue;
        p[u].load((const char*)t.p + o * (PBF ? 2 : 4), lane, left);
        g[u].load((const char*)t.g + o * (GBF ? 2 : 4), lane, left);
        if (BITS8) {
            qm[u] = load_codes<FULL>((const uint8_t*)t.m + o, lane, left);
            qv[u] = load_codes<FULL>((const uint8_t*)t.v + o, lane, left);
            ee[u] = (uint32_t)t.e[2 * (o / kBlock)] | (uint32_t)t.e[2 * (o / kBlock) + 1] << 16;
        } else {
            fm[u].load((const float*)t.m + o, lane, left);
            fv[u].load((const float*)t.v + o, lane, left);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t o = base + u * stride;
        const int left = left0 - u * stride;
        if (!FULL && left <= 0) continue;
        float m[4], v[4];
        if (BITS8) {
            const float sm = __uint_as_float((ee[u] & 0xFFu) << 23), sv = __uint_as_float((ee[u] >> 16) << 23);
            const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)qm[u], false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)qm[u], true);
            const auto v01 = __builtin_amdgcn_cvt_pk_f32_bf8((int)qv[u], false), v23 = __builtin_amdgcn_cvt_pk_f32_bf8((int)qv[u], true);
            m[0] = m01[0] * sm; m[1] = m01[1] * sm; m[2] = m23[0] * sm; m[3] = m23[1] * sm;
            v[0] = v01[0] * sv; v[1] = v01[1] * sv; v[2] = v23[0] * sv; v[3] = v23[1] * sv;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) { m[j] = fm[u].get(j); v[j] = fv[u].get(j); }
        }
        Four<true, FULL> copy;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float gj = g[u].get(j) * s.gs, pj = p[u].get(j);
            m[j] = m[j] * a.b1 + gj * a.omb1;
            v[j] = v[j] * a.b2 + gj * gj * a.omb2;
            const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[j]) * s.rc2 + a.eps);
            p[u].set(j, pj - (s.step * m[j] * r + s.decay * pj));
            copy.set(j, p[u].get(j));
        }
        p[u].store((char*)t.p + o * (PBF ? 2 : 4), lane, left);
        if (t.copy) copy.store(t.copy + o, lane, left);
        if (!BITS8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { fm[u].set(j, m[j]); fv[u].set(j, v[j]); }
            fm[u].store((float*)t.m + o, lane, left);
            fv[u].store((float*)t.v + o, lane, left);
            continue;
        }
        uint32_t mm = 0, mv = 0, bad = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (behind the end the loads gave zeros, and zeros they stay)
            const uint32_t um = __float_as_uint(m[j]) & 0x7FFFFFFFu, uv = __float_as_uint(v[j]) & 0x7FFFFFFFu;
            if (um < 0x7F800000u) mm = mm > um ? mm : um; else bad = 1;
            if (uv < 0x7F800000u) mv = mv > uv ? mv : uv; else bad = 1;
        }
        const int em = block_exponent<8>(wave_max(mm)), ev = block_exponent<15>(wave_max(mv));
        const float im = __uint_as_float((uint32_t)(254 - em) << 23), iv = __uint_as_float((uint32_t)(254 - ev) << 23);
        uint32_t om = 0, ov = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t c = t.first + (uint64_t)o + (uint64_t)(4 * lane + j);
            const uint32_t r = odw_mix(odw_mix((uint32_t)c ^ a.k0) + s.k1 + (uint32_t)(c >> 32));
            om |= encode8<7, 3>(m[j], im, r & 0xFFFFu, 0, bad) << (8 * j);
            ov |= encode8<15, 2>(v[j], iv, r >> 16, s.least_v, bad) << (8 * j);
        }
        store_codes<FULL>((uint8_t*)t.m + o, lane, left, om);
        store_codes<FULL>((uint8_t*)t.v + o, lane, left, ov);
        if (lane == 0) {
            t.e[2 * (o / kBlock)] = (uint8_t)em;
            t.e[2 * (o / kBlock) + 1] = (uint8_t)ev;
        }
    }
}

// A chunk: its four waves take every fourth block, all at once -- a tensor's last, short chunk as well, whose blocks one after the other
// would cost small tensors a round trip to memory each.
template <bool BITS8, bool PBF, bool GBF>
__device__ __forceinline__ void chunk(const Args& a, const Tensor& t, const Step& s, int64_t begin, int wave, int lane) {
    constexpr int kWaves = kThreads / 64;
    const int64_t rest = t.n - begin, base = begin + wave * kBlock;
    if (rest >= chunk_of(BITS8)) update<BITS8, PBF, GBF, true, unroll(BITS8)>(a, t, s, base, kWaves * kBlock, lane, 0);
    else update<BITS8, PBF, GBF, false, unroll(BITS8)>(a, t, s, base, kWaves * kBlock, lane, (int)rest - wave * kBlock);
}

template <bool BITS8>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Args a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float c1 = a.c1, c2 = a.c2;
    Step s;
    s.k1 = a.k1;
    if (a.bias) {
        c1 = a.bias[0];
        c2 = a.bias[1];
        s.k1 += __float_as_uint(a.bias[2]);        // the step's number: a replayed launch draws new bits
    }
    s.gs = a.scale ? a.mult * *a.scale : a.mult;
    s.rc2 = 1.0f / sqrtf(c2);
    const Prefix<kMaxTensors> prefix(a.chunk0, a.count);
    for (int c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const int ti = prefix.tensor_of(c);
        const Tensor& t = a.t[ti];
        const int64_t begin = (int64_t)(c - prefix.chunk0_of(ti)) * chunk_of(BITS8);
        s.step = t.lr / c1;
        s.decay = t.lr * t.wd;
        s.least_v = t.flags & kVToZero ? 0 : 1;
        switch (t.flags & (kPBf16 | kGBf16)) {     // (a tensor's types: uniform)
            case 0: chunk<BITS8, false, false>(a, t, s, begin, wave, lane); break;
            case kPBf16: chunk<BITS8, true, false>(a, t, s, begin, wave, lane); break;
            case kGBf16: chunk<BITS8, false, true>(a, t, s, begin, wave, lane); break;
            default: chunk<BITS8, true, true>(a, t, s, begin, wave, lane); break;
        }
    }
}

// step += 1 on the device, and what the update needs of it: the bias corrections and the step's low word.
__global__ void adamw_advance_kernel(int64_t* step, double b1, double b2, float* bias) {
    const int64_t t = *step + 1;
    *step = t;
    bias[0] = (float)(1.0 - pow(b1, (double)t));
    bias[1] = (float)(1.0 - pow(b2, (double)t));
    bias[2] = __uint_as_float((uint32_t)t);
}

// ---- the global norm ------------------------------------------------------------------------------------------------------------
// Sum of squares of a chunk: fp32 products exact in fp64, summed in fp64 in a fixed order.
template <bool BF>
__device__ __forceinline__ double sqsum(const void* g, int size, int wave, int lane) {
    constexpr int kWaves = kThreads / 64, U = 8;
    const int blocks = size / kBlock;
    double s = 0.0;
    int b = wave;
    for (; b + (U - 1) * kWaves < blocks; b += U * kWaves) {
        Four<BF, true> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].load((const char*)g + (size_t)(b + u * kWaves) * kBlock * (BF ? 2 : 4), lane, kBlock);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) s = fma((double)x[u].get(j), (double)x[u].get(j), s);
    }
    for (; b * kBlock < size; b += U * kWaves) {
        Four<BF, false> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            x[u].load((const char*)g + (size_t)(b + u * kWaves) * kBlock * (BF ? 2 : 4), lane, size - (b + u * kWaves) * kBlock);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) s = fma((double)x[u].get(j), (double)x[u].get(j), s);
    }
    return s;
}

__global__ __launch_bounds__(kThreads) void sqsum_kernel(const NormArgs a, double* __restrict__ partial) {
    __shared__ double part[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = blockIdx.x;
    const Prefix<kNormTensors> prefix(a.chunk0, a.count);
    const int ti = prefix.tensor_of(c);
    const int64_t begin = (int64_t)(c - prefix.chunk0_of(ti)) * kNormChunk, rest = a.n[ti] - begin;
    const int size = rest < kNormChunk ? (int)rest : kNormChunk;
    const bool bf = a.flags[ti] & kGBf16;
    const char* g = (const char*)a.g[ti] + begin * (bf ? 2 : 4);
    double s = bf ? sqsum<true>(g, size, wave, lane) : sqsum<false>(g, size, wave, lane);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) part[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[c] = part[0] + part[1] + part[2] + part[3];
}

// out[0] = sqrt(sum of the partial sums), out[1] = min(1, max_norm / (norm + 1e-6)) (NaN stays NaN).
__global__ __launch_bounds__(1024) void norm_finish_kernel(const double* __restrict__ partial, int count, double max_norm,
                                                           float* __restrict__ out) {
    __shared__ double part[16];
    double s = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += 1024) s += partial[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; ++i) t += part[i];
        const double norm = sqrt(t), c = max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = c > 1.0 ? 1.0f : (float)c;
    }
}

template <bool BF>
__device__ __forceinline__ void scale(void* g, int size, int wave, int lane, float s) {
    constexpr int kWaves = kThreads / 64, U = 4;
    const int blocks = size / kBlock;
    int b = wave;
    for (; b + (U - 1) * kWaves < blocks; b += U * kWaves) {
        Four<BF, true> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].load((const char*)g + (size_t)(b + u * kWaves) * kBlock * (BF ? 2 : 4), lane, kBlock);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u].set(j, x[u].get(j) * s);
            x[u].store((char*)g + (size_t)(b + u * kWaves) * kBlock * (BF ? 2 : 4), lane, kBlock);
        }
    }
    for (; b * kBlock < size; b += kWaves) {
        Four<BF, false> x;
        x.load((const char*)g + (size_t)b * kBlock * (BF ? 2 : 4), lane, size - b * kBlock);
#pragma unroll
        for (int j = 0; j < 4; ++j) x.set(j, x.get(j) * s);
        x.store((char*)g + (size_t)b * kBlock * (BF ? 2 : 4), lane, size - b * kBlock);
    }
}

__global__ __launch_bounds__(kThreads) void scale_kernel(const NormArgs a, const float* __restrict__ factor) {
    const float s = *factor;
    if (s == 1.0f) return;                       // the products would be what is there
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = blockIdx.x;
    const Prefix<kNormTensors> prefix(a.chunk0, a.count);
    const int ti = prefix.tensor_of(c);
    const int64_t begin = (int64_t)(c - prefix.chunk0_of(ti)) * kNormChunk, rest = a.n[ti] - begin;
    const int size = rest < kNormChunk ? (int)rest : kNormChunk;
    const bool bf = a.flags[ti] & kGBf16;
    char* g = (char*)const_cast<void*>(a.g[ti]) + begin * (bf ? 2 : 4);
    if (bf) scale<true>(g, size, wave, lane, s);
    else scale<false>(g, size, wave, lane, s);
}

bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
int64_t chunks_of(int64_t n, int chunk) { return (n + chunk - 1) / chunk; }
constexpr int64_t kMaxElements = (int64_t)1 << 40;           // of one tensor: its chunks fit an int

// Fills `a` with tensors from `i` on (empty ones left out) until it is full; returns the first one not taken.
int fill_norm_args(NormArgs& a, int i, int n_tensors, const void* const* g, const int64_t* n, const int* types) {
    a.count = a.chunks = 0;
    for (; i < n_tensors && a.count < kNormTensors; ++i) {
        if (n[i] == 0) continue;
        if (a.count && a.chunks + chunks_of(n[i], kNormChunk) > INT32_MAX) break;
        a.g[a.count] = g[i];
        a.n[a.count] = n[i];
        a.flags[a.count] = (uint8_t)(types[i] & kGBf16);
        a.chunk0[a.count] = a.chunks;
        a.chunks += (int)chunks_of(n[i], kNormChunk);
        ++a.count;
    }
    return i;
}

int check_list(const char* what, int n_tensors, const void* const* g, const int64_t* n, const int* types, int all_types = kPBf16 | kGBf16) {
    ODW_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || (g && n && types)), "%s: null list", what);
    for (int i = 0; i < n_tensors; ++i) {
        ODW_REQUIRE(n[i] >= 0 && n[i] < kMaxElements, "%s: tensor %d has %lld elements", what, i, (long long)n[i]);
        ODW_REQUIRE(n[i] == 0 || g[i], "%s: tensor %d: null pointer", what, i);
        ODW_REQUIRE(types[i] >= 0 && types[i] <= all_types, "%s: tensor %d: bad type %d", what, i, types[i]);
        ODW_REQUIRE(aligned(g[i], types[i] & kGBf16 ? 2 : 4), "%s: tensor %d: pointer not aligned to its elements", what, i);
    }
    return ODW_OK;
}

int adamw(bool bits8, int n_tensors, void* const* p, const void* const* g, void* const* m, void* const* v, uint8_t* const* e,
          void* const* copy, const int64_t* n, const int* types, const float* lr, const float* wd, double beta1, double beta2,
          double eps, int64_t step, const float* bias, const float* grad_scale, float grad_mult, uint32_t k0, uint32_t k1,
          int max_workgroups, hipStream_t stream) {
    const char* what = bits8 ? "adamw8" : "adamw";
    const int rc = check_list(what, n_tensors, g, n, types, kPBf16 | kGBf16 | (bits8 ? kVToZero : 0));
    if (rc != ODW_OK) return rc;
    ODW_REQUIRE(n_tensors == 0 || (p && m && v && lr && wd && (!bits8 || e)), "%s: null list", what);
    ODW_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "%s: betas %g, %g not in [0, 1)", what, beta1, beta2);
    ODW_REQUIRE(eps >= 1e-15, "%s: eps %g is under 1e-15 (squares of gradients underflow before they are small beside it)", what, eps);
    ODW_REQUIRE(bias || step >= 1, "%s: step %lld is not positive", what, (long long)step);
    ODW_REQUIRE(max_workgroups >= 0, "%s: max_workgroups %d", what, max_workgroups);
    for (int i = 0; i < n_tensors; ++i) {
        if (n[i] == 0) continue;
        ODW_REQUIRE(p[i] && m[i] && v[i] && (!bits8 || e[i]), "%s: tensor %d: null pointer", what, i);
        ODW_REQUIRE(aligned(p[i], types[i] & kPBf16 ? 2 : 4) && (!copy || aligned(copy[i], 2)) &&
                        (bits8 || (aligned(m[i], 4) && aligned(v[i], 4))), "%s: tensor %d: pointer not aligned to its elements", what, i);
    }
    Args a;
    a.b1 = (float)beta1; a.b2 = (float)beta2; a.omb1 = (float)(1.0 - beta1); a.omb2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.c1 = bias ? 1.0f : (float)(1.0 - pow(beta1, (double)step));
    a.c2 = bias ? 1.0f : (float)(1.0 - pow(beta2, (double)step));
    // keys that differ in k0 alone would permute one set of numbers over the elements (the hash starts from counter ^ k0): a small
    // tensor would meet the same few thousand numbers step after step, and their excess over the mean would not average out
    a.mult = grad_mult; a.k0 = k0; a.k1 = k1 + 0x9E3779B9u * k0; a.scale = grad_scale; a.bias = bias;
    uint64_t first = 0;
    for (int i = 0; i < n_tensors;) {
        a.count = a.chunks = 0;
        for (; i < n_tensors && a.count < kMaxTensors; ++i) {
            if (n[i] == 0) continue;
            if (a.count && a.chunks + chunks_of(n[i], chunk_of(bits8)) > INT32_MAX) break;
            a.chunk0[a.count] = a.chunks;
            Tensor& t = a.t[a.count++];
            t.p = p[i]; t.g = g[i]; t.m = m[i]; t.v = v[i]; t.e = bits8 ? e[i] : nullptr;
            t.copy = copy ? (unsigned short*)copy[i] : nullptr;
            t.n = n[i]; t.first = first; t.lr = lr[i]; t.wd = wd[i];
            t.flags = types[i];
            a.chunks += (int)chunks_of(n[i], chunk_of(bits8));
            first += (uint64_t)n[i];
        }
        if (!a.count) break;
        const int most = max_workgroups > 0 && max_workgroups < kMaxGrid ? max_workgroups : kMaxGrid;
        const int grid = a.chunks < most ? a.chunks : most;
        if (bits8) adamw_kernel<true><<<grid, kThreads, 0, stream>>>(a);
        else adamw_kernel<false><<<grid, kThreads, 0, stream>>>(a);
        ODW_CHECK_LAUNCH("adamw_kernel");
    }
    return ODW_OK;
}

}  // namespace

ODW_EXPORT int64_t odw_grad_norm_workspace(int n_tensors, const int64_t* n) {
    int64_t chunks = 0;
    for (int i = 0; i < n_tensors; ++i) chunks += n[i] > 0 ? chunks_of(n[i], kNormChunk) : 0;
    return chunks * (int64_t)sizeof(double);
}

ODW_EXPORT int odw_grad_norm(int n_tensors, const void* const* g, const int64_t* n, const int* types, double max_norm, float* out,
                             void* workspace, int64_t workspace_bytes, void* stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const int rc = check_list("grad_norm", n_tensors, g, n, types);
    if (rc != ODW_OK) return rc;
    ODW_REQUIRE(out, "grad_norm: null output");
    ODW_REQUIRE(max_norm > 0.0, "grad_norm: max_norm %g is not positive", max_norm);
    const int64_t need = odw_grad_norm_workspace(n_tensors, n);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        odw_set_error("grad_norm: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
        return ODW_EWORKSPACE;
    }
    ODW_REQUIRE(aligned(workspace, 8), "grad_norm: workspace must be 8-byte aligned");
    ODW_REQUIRE(need / (int64_t)sizeof(double) <= INT32_MAX, "grad_norm: too many elements");
    NormArgs a;
    int done = 0;
    for (int i = 0; i < n_tensors;) {
        i = fill_norm_args(a, i, n_tensors, g, n, types);
        if (!a.count) break;
        sqsum_kernel<<<a.chunks, kThreads, 0, stream>>>(a, (double*)workspace + done);
        ODW_CHECK_LAUNCH("sqsum_kernel");
        done += a.chunks;
    }
    norm_finish_kernel<<<1, 1024, 0, stream>>>((const double*)workspace, done, max_norm, out);
    ODW_CHECK_LAUNCH("norm_finish_kernel");
    return ODW_OK;
}

ODW_EXPORT int odw_scale_tensors(int n_tensors, void* const* x, const int64_t* n, const int* types, const float* scale, void* stream_) {
    const int rc = check_list("scale_tensors", n_tensors, x, n, types);
    if (rc != ODW_OK) return rc;
    ODW_REQUIRE(scale, "scale_tensors: null scale");
    NormArgs a;
    for (int i = 0; i < n_tensors;) {
        i = fill_norm_args(a, i, n_tensors, x, n, types);
        if (!a.count) break;
        scale_kernel<<<a.chunks, kThreads, 0, (hipStream_t)stream_>>>(a, scale);
        ODW_CHECK_LAUNCH("scale_kernel");
    }
    return ODW_OK;
}

ODW_EXPORT int odw_adamw_advance(int64_t* step, double beta1, double beta2, float* bias, void* stream_) {
    ODW_REQUIRE(step && bias, "adamw_advance: null pointer");
    adamw_advance_kernel<<<1, 1, 0, (hipStream_t)stream_>>>(step, beta1, beta2, bias);
    ODW_CHECK_LAUNCH("adamw_advance_kernel");
    return ODW_OK;
}

ODW_EXPORT int odw_adamw(int n_tensors, void* const* p, const void* const* g, void* const* m, void* const* v, void* const* copy,
                         const int64_t* n, const int* types, const float* lr, const float* wd, double beta1, double beta2, double eps,
                         int64_t step, const float* bias, const float* grad_scale, float grad_mult, int max_workgroups, void* stream_) {
    return adamw(false, n_tensors, p, g, m, v, nullptr, copy, n, types, lr, wd, beta1, beta2, eps, step, bias, grad_scale, grad_mult, 0,
                 0, max_workgroups, (hipStream_t)stream_);
}

ODW_EXPORT int odw_adamw8(int n_tensors, void* const* p, const void* const* g, void* const* m, void* const* v, uint8_t* const* e,
                          void* const* copy, const int64_t* n, const int* types, const float* lr, const float* wd, double beta1,
                          double beta2, double eps, int64_t step, const float* bias, const float* grad_scale, float grad_mult,
                          uint32_t k0, uint32_t k1, int max_workgroups, void* stream_) {
    return adamw(true, n_tensors, p, g, m, v, e, copy, n, types, lr, wd, beta1, beta2, eps, step, bias, grad_scale, grad_mult, k0, k1,
                 max_workgroups, (hipStream_t)stream_);
}
