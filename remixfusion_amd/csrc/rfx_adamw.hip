// rfx_adamw.hip -- AdamW over many tensors (moments in 32 or in 8 bits), the gradients' global norm and their scaling.
//
// Every kernel here is one pass over its data: an element of the step costs 28 bytes (fp32 parameter, 32-bit moments) or 16
// (8-bit moments) of HBM traffic and some dozens of vector instructions, so the bytes are the bound and the instructions are
// what has to stay under them.  All tensors of a kind (type, state, master copy) go into one launch: their descriptors travel in
// the kernel's arguments (no table in device memory that a later call could overwrite under a running kernel or a captured one),
// every tensor is cut into pieces of PIECE elements, and a block finds its tensor by bisection over the first pieces.
#include "rfx_common.h"
#include <math.h>

namespace rfx {

constexpr int AW_THREADS = 256;
constexpr int AW_PIECE = 4096;          // elements per block
constexpr int AW_TENSORS = 48;          // descriptors per launch: the kernel's arguments stay under 4 KB
constexpr int AW_GROUPS = 8;
constexpr int AW_RUN = RFX_ADAMW_BLOCK;

struct AwTensor {
    void* p;
    const void* g;
    void* m;
    void* v;
    int8_t* e;
    float* w;
    int64_t n;
    int32_t group;
    uint32_t index;
};

// what the step count decides; per group from the host, or per tensor from adamw_prepare_kernel
struct AwStep {
    float step_size;                    // lr / (1 - b1^k)
    float inv_bc2;                      // 1 / sqrt(1 - b2^k)
    float lr_wd;
    uint32_t key;                       // hash of (seed, k)
};

struct AwGroup {
    double b1, c1, b2, c2;              // beta, 1 - beta
    AwStep s;
    float eps;
    float sign;                         // -1: maximize
};

struct AwArgs {
    AwTensor t[AW_TENSORS];
    int32_t first[AW_TENSORS + 1];
    AwGroup group[AW_GROUPS];
    const AwStep* dev;                  // per tensor of this launch, or null
    const double* clip;
    int32_t count;
};
static_assert(sizeof(AwArgs) <= 4096, "kernel arguments");

template <int TYPE> struct Elem;
template <> struct Elem<RFX_F32> { typedef float T; };
template <> struct Elem<RFX_BF16> { typedef __bf16 T; };
template <> struct Elem<RFX_F16> { typedef _Float16 T; };
template <typename T> using vec4 = T __attribute__((ext_vector_type(4)));
typedef vec4<float> f4;

__device__ __forceinline__ f4 widen(vec4<float> x) { return x; }
__device__ __forceinline__ f4 widen(vec4<__bf16> x) { return __builtin_convertvector(x, f4); }
__device__ __forceinline__ f4 widen(vec4<_Float16> x) { return __builtin_convertvector(x, f4); }

template <typename T> __device__ __forceinline__ f4 load4(const T* p) { return widen(*reinterpret_cast<const vec4<T>*>(p)); }
template <typename T> __device__ __forceinline__ void store4(T* p, f4 x) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f4*>(p) = x;
    else *reinterpret_cast<vec4<T>*>(p) = __builtin_convertvector(x, vec4<T>);      // to nearest, ties to even: once, at the end
}

// xor-shift / multiply mixer of 32-bit integers (a bijection)
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7feb352dU;
    x ^= x >> 15; x *= 0x846ca68bU;
    return x ^ (x >> 16);
}

// which tensor a piece belongs to: the last one whose first piece is not behind it
__device__ __forceinline__ int find(const int32_t* first, int count, int piece) {
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= piece) lo = mid; else hi = mid;
    }
    return lo;
}

__host__ __device__ inline AwStep step_scalars(double lr, double b1, double b2, double wd, double k, uint32_t seed) {
    AwStep s;
    s.step_size = (float)(lr / (1.0 - pow(b1, k)));
    s.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(b2, k)));
    s.lr_wd = (float)(lr * wd);
    s.key = mix32(mix32(seed) + (uint32_t)(int64_t)k);
    return s;
}

// p - (lr wd p + step_size m / (sqrt(v) / sqrt(1 - b2^k) + eps)): the two small terms meet before they meet p, so a decay of less
// than half a unit of p's last place is not lost to a rounding of its own
__device__ __forceinline__ float stepped(float p, float m, float v, const AwStep& s, float eps) {
    const float d = madd(sqrtf(v), s.inv_bc2, eps);
    return p - madd(s.lr_wd, p, s.step_size * (m / d));
}

// ---- 32-bit moments: fp32 throughout ------------------------------------------------------------------------------------------
__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, const AwGroup& a, const AwStep& s, float c) {
    const float c1 = (float)a.c1, c2 = (float)a.c2, b1 = (float)a.b1, b2 = (float)a.b2;
    g *= c;
    m = madd(c1, g, b1 * m);
    v = madd(c2 * g, g, b2 * v);
    p = stepped(p, m, v, s, a.eps);
}

template <int TYPE, bool MASTER>
__global__ __launch_bounds__(AW_THREADS) void adamw32_kernel(const AwArgs k) {
    typedef typename Elem<TYPE>::T T;
    const int ti = find(k.first, k.count, (int)blockIdx.x);
    const AwTensor& t = k.t[ti];
    const AwGroup& a = k.group[t.group];
    const AwStep s = k.dev ? k.dev[ti] : a.s;
    const float c = a.sign * (k.clip ? (float)k.clip[1] : 1.f);
    const int64_t base = (int64_t)((int)blockIdx.x - k.first[ti]) * AW_PIECE;
    const int len = (int)(t.n - base < AW_PIECE ? t.n - base : AW_PIECE);
    T* p = (T*)t.p + base;
    const T* g = (const T*)t.g + base;
    float* m = (float*)t.m + base;
    float* v = (float*)t.v + base;
    float* w = MASTER ? t.w + base : nullptr;
    const bool vec = ((((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) | (((uintptr_t)m | (uintptr_t)v | (uintptr_t)w) & 15)) == 0;
    int done = 0;
    if (vec) {
        done = len & ~3;
        for (int i = threadIdx.x * 4; i < done; i += AW_THREADS * 4) {
            f4 x = MASTER ? load4(w + i) : load4(p + i);
            const f4 gg = load4(g + i);
            f4 mm = load4(m + i), vv = load4(v + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float xj = x[j], mj = mm[j], vj = vv[j];
                adamw_one(xj, gg[j], mj, vj, a, s, c);
                x[j] = xj; mm[j] = mj; vv[j] = vj;
            }
            store4(p + i, x);
            if (MASTER) store4(w + i, x);
            store4(m + i, mm);
            store4(v + i, vv);
        }
    }
    for (int i = done + threadIdx.x; i < len; i += AW_THREADS) {
        float x = MASTER ? w[i] : (float)p[i], mm = m[i], vv = v[i];
        adamw_one(x, (float)g[i], mm, vv, a, s, c);
        p[i] = (T)x;
        if (MASTER) w[i] = x;
        m[i] = mm; v[i] = vv;
    }
}

// ---- 8-bit moments ------------------------------------------------------------------------------------------------------------
// A wave owns a run of 256 elements, four consecutive ones a lane.  The moments are formed in fp64 (full rate on this chip), so
// that which side of a border they fall on does not depend on the order of the operations; the update is fp32.
//   decode: a byte's seven (eight) bits moved to an fp32's exponent and mantissa ARE the format, subnormals included, times a power
//           of two that is a constant of the run;
//   encode: the moment times the inverse power of two, rounded to fp32 (subnormals included), leaves 20 bits below the format's
//           last place: 16 random bits (and half of their unit) are added, and the upper bits are the code.
__device__ __forceinline__ double pow2(int e) { return __longlong_as_double((long long)(e + 1023) << 52); }

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t y = (uint32_t)__shfl_xor((int)x, d, 64);
        x = x > y ? x : y;
    }
    return x;
}

// exponent byte of a run from the upper word of its largest magnitude (an fp64's bits order like integers, NaN above all).
// UNIT 2: second moments, squares of fp32 numbers, span twice the exponents that a byte has, so theirs count in twos
template <int UNIT> __device__ __forceinline__ int run_exponent(uint32_t hi) {
    if (hi >= 0x7ff00000U) return -128;
    int e = (int)((hi + (1U << 17)) >> 20) - 1023;                     // the addition carries where the significand is >= 1.875
    if (UNIT == 2) e = (e + 1) >> 1;
    return e < -127 ? -127 : e > 127 ? 127 : e;
}

__device__ __forceinline__ double scale_m(int byte) { return byte == -128 ? __builtin_nan("") : pow2(byte + 112); }
__device__ __forceinline__ double scale_v(int byte) { return byte == -128 ? __builtin_nan("") : pow2(2 * byte + 96); }

template <int TOP> __device__ __forceinline__ uint32_t encode(double mag, double inverse, uint32_t r16) {
    const uint32_t z = __float_as_uint((float)(mag * inverse)) + (r16 << 4) + 8;
    const uint32_t c = z >> 20;
    return c < (uint32_t)TOP ? c : (uint32_t)TOP;
}

template <int TYPE, bool MASTER>
__global__ __launch_bounds__(AW_THREADS) void adamw8_kernel(const AwArgs k) {
    typedef typename Elem<TYPE>::T T;
    const int ti = find(k.first, k.count, (int)blockIdx.x);
    const AwTensor& t = k.t[ti];
    const AwGroup& a = k.group[t.group];
    const AwStep s = k.dev ? k.dev[ti] : a.s;
    const double c = (double)a.sign * (k.clip ? k.clip[1] : 1.0);
    const int64_t piece = (int)blockIdx.x - k.first[ti];
    const int64_t base = piece * AW_PIECE;
    const int len = (int)(t.n - base < AW_PIECE ? t.n - base : AW_PIECE);
    const int64_t runs = (t.n + AW_RUN - 1) / AW_RUN;
    const uint32_t key = mix32(s.key + t.index);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* g = (const T*)t.g + base;
    T* p = (T*)t.p + base;
    float* w = MASTER ? t.w + base : nullptr;
    uint8_t* m = (uint8_t*)t.m + base;
    uint8_t* v = (uint8_t*)t.v + base;
    const bool vec = ((((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) | ((uintptr_t)w & 15)) == 0;
    for (int r = wave; r * AW_RUN < len; r += AW_THREADS / 64) {
        const int64_t run = piece * (AW_PIECE / AW_RUN) + r;
        const int i = r * AW_RUN + lane * 4;
        const int have = len - i < 0 ? 0 : len - i > 4 ? 4 : len - i;  // elements of this lane
        f4 x = {0, 0, 0, 0}, gg = {0, 0, 0, 0};
        uint32_t cm = 0, cv = 0;
        if (have == 4 && vec) {
            x = MASTER ? load4(w + i) : load4(p + i);
            gg = load4(g + i);
        } else {
            for (int j = 0; j < have; ++j) { x[j] = MASTER ? w[i + j] : (float)p[i + j]; gg[j] = (float)g[i + j]; }
        }
        if (have == 4) {
            cm = *reinterpret_cast<const uint32_t*>(m + i);
            cv = *reinterpret_cast<const uint32_t*>(v + i);
        } else {
            for (int j = 0; j < have; ++j) { cm |= (uint32_t)m[i + j] << (8 * j); cv |= (uint32_t)v[i + j] << (8 * j); }
        }
        const double s1 = scale_m(t.e[run]), s2 = scale_v(t.e[runs + run]);
        double md[4], vd[4];
        uint32_t h1 = 0, h2 = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t bm = (cm >> (8 * j)) & 255, bv = (cv >> (8 * j)) & 255;
            const double gd = (double)gg[j] * c;
            md[j] = (double)__uint_as_float((bm & 127) << 20 | (bm & 128) << 24) * s1 * a.b1 + gd * a.c1;
            vd[j] = (double)__uint_as_float(bv << 20) * s2 * a.b2 + gd * gd * a.c2;
            const uint32_t u1 = (uint32_t)__double2hiint(md[j]) & 0x7fffffffU, u2 = (uint32_t)__double2hiint(vd[j]) & 0x7fffffffU;
            if (j < have) { h1 = h1 > u1 ? h1 : u1; h2 = h2 > u2 ? h2 : u2; }
        }
        const int n1 = run_exponent<1>(wave_max(h1)), n2 = run_exponent<2>(wave_max(h2));
        const double i1 = pow2(-112 - n1), i2 = pow2(-96 - 2 * n2);
        const uint32_t hash = mix32(key + (uint32_t)run);
        cm = 0; cv = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t r16 = mix32(hash + (uint32_t)(lane * 4 + j) * 0x9e3779b9U);
            uint32_t bm = encode<127>(fabs(md[j]), i1, r16 & 0xffff), bv = encode<255>(vd[j], i2, r16 >> 16);
            if (vd[j] > 0.0 && bv == 0) bv = 1;
            if (n1 == -128) bm = 0;
            if (n2 == -128) bv = 0;
            bm |= md[j] < 0.0 ? 128 : 0;
            cm |= bm << (8 * j);
            cv |= bv << (8 * j);
            x[j] = stepped(x[j], (float)md[j], (float)vd[j], s, a.eps);
        }
        if (have == 4 && vec) {
            store4(p + i, x);
            if (MASTER) store4(w + i, x);
        } else {
            for (int j = 0; j < have; ++j) { p[i + j] = (T)x[j]; if (MASTER) w[i + j] = x[j]; }
        }
        if (have == 4) {
            *reinterpret_cast<uint32_t*>(m + i) = cm;
            *reinterpret_cast<uint32_t*>(v + i) = cv;
        } else {
            for (int j = 0; j < have; ++j) { m[i + j] = (uint8_t)(cm >> (8 * j)); v[i + j] = (uint8_t)(cv >> (8 * j)); }
        }
        if (lane == 0) { t.e[run] = (int8_t)n1; t.e[runs + run] = (int8_t)n2; }
    }
}

// step counts on the device (captured calls): raise them and derive what they decide, one thread a tensor
struct PrepArgs {
    float* step[AW_TENSORS];
    uint8_t group[AW_TENSORS];
    struct { double lr, b1, b2, wd; const float* lr_dev; uint32_t seed; } g[AW_GROUPS];
    AwStep* out;
    int32_t count;
};
static_assert(sizeof(PrepArgs) <= 4096, "kernel arguments");

__global__ __launch_bounds__(64) void adamw_prepare_kernel(const PrepArgs k) {
    const int i = threadIdx.x;
    if (i >= k.count) return;
    const auto& g = k.g[k.group[i]];
    const float step = *k.step[i] + 1.f;
    *k.step[i] = step;
    k.out[i] = step_scalars(g.lr_dev ? (double)*g.lr_dev : g.lr, g.b1, g.b2, g.wd, (double)step, g.seed);
}

// ---- fp32 values of 8-bit moments -----------------------------------------------------------------------------------------------
struct MomArgs {
    rfx_moment_tensor t[AW_TENSORS];
    int32_t first[AW_TENSORS + 1];
    int32_t count;
};
static_assert(sizeof(MomArgs) <= 4096, "kernel arguments");

__global__ __launch_bounds__(AW_THREADS) void adamw_moments_kernel(const MomArgs k) {
    const int ti = find(k.first, k.count, (int)blockIdx.x);
    const rfx_moment_tensor& t = k.t[ti];
    const int64_t piece = (int)blockIdx.x - k.first[ti], base = piece * AW_PIECE;
    const int len = (int)(t.n - base < AW_PIECE ? t.n - base : AW_PIECE);
    const int64_t runs = (t.n + AW_RUN - 1) / AW_RUN;
    const uint8_t* m = t.exp_avg + base;
    const uint8_t* v = t.exp_avg_sq + base;
    float* om = t.out_avg + base;
    float* ov = t.out_avg_sq + base;
    const bool vec = (((uintptr_t)om | (uintptr_t)ov) & 15) == 0;
    for (int i = threadIdx.x * 4; i < len; i += AW_THREADS * 4) {
        const int64_t run = piece * (AW_PIECE / AW_RUN) + i / AW_RUN;
        const int have = len - i > 4 ? 4 : len - i;
        const double s1 = scale_m(t.exponents[run]), s2 = scale_v(t.exponents[runs + run]);
        uint32_t cm = 0, cv = 0;
        if (have == 4) {
            cm = *reinterpret_cast<const uint32_t*>(m + i);
            cv = *reinterpret_cast<const uint32_t*>(v + i);
        } else {
            for (int j = 0; j < have; ++j) { cm |= (uint32_t)m[i + j] << (8 * j); cv |= (uint32_t)v[i + j] << (8 * j); }
        }
        f4 a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t bm = (cm >> (8 * j)) & 255, bv = (cv >> (8 * j)) & 255;
            a[j] = (float)((double)__uint_as_float((bm & 127) << 20 | (bm & 128) << 24) * s1);
            b[j] = (float)((double)__uint_as_float(bv << 20) * s2);
        }
        if (have == 4 && vec) {
            store4(om + i, a);
            store4(ov + i, b);
        } else {
            for (int j = 0; j < have; ++j) { om[i + j] = a[j]; ov[i + j] = b[j]; }
        }
    }
}

// ---- global norm ------------------------------------------------------------------------------------------------------------
constexpr int GN_TENSORS = 128;
constexpr int GN_THREADS = 256;
constexpr int GN_PIECE = 16384;
constexpr int GN_BLOCKS = 1024;         // partial sums of a launch at most

struct GnArgs {
    struct { void* g; int64_t n; } t[GN_TENSORS];
    int32_t first[GN_TENSORS + 1];
    uint8_t dtype[GN_TENSORS];
    double* partial;
    const double* clip;
    int32_t count, pieces, kind;
};
static_assert(sizeof(GnArgs) <= 4096, "kernel arguments");

template <typename T, bool MAX> __device__ __forceinline__ void norm_piece(const T* g, int len, double& sum, uint32_t& big) {
    int done = 0;
    auto one = [&](float x) {
        if (MAX) { const uint32_t u = __float_as_uint(x) & 0x7fffffffU; big = big > u ? big : u; }      // integers order NaN above all
        else { const double d = (double)x; sum = fma(d, d, sum); }
    };
    if (((uintptr_t)g & (4 * sizeof(T) - 1)) == 0) {
        done = len & ~3;
        for (int i = threadIdx.x * 4; i < done; i += GN_THREADS * 4) {
            const f4 x = load4(g + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) one(x[j]);
        }
    }
    for (int i = done + threadIdx.x; i < len; i += GN_THREADS) one((float)g[i]);
}

__device__ __forceinline__ double block_sum(double x, double* lds) {       // every thread gets the sum; fixed order
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < GN_THREADS / 64; ++w) s += lds[w];
    return s;
}

__device__ __forceinline__ double block_max(double x, double* lds) {       // of non-negative values; NaN wins
    const auto larger = [](double p, double q) { return p != p ? p : (q != q || q > p) ? q : p; };
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x = larger(x, __shfl_xor(x, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < GN_THREADS / 64; ++w) s = larger(s, lds[w]);
    return s;
}

template <bool MAX>
__global__ __launch_bounds__(GN_THREADS) void grad_norm_kernel(const GnArgs k) {
    __shared__ double lds[GN_THREADS / 64];
    double sum = 0.0;
    uint32_t big = 0;
    for (int piece = blockIdx.x; piece < k.pieces; piece += gridDim.x) {
        const int ti = find(k.first, k.count, piece);
        const int64_t base = (int64_t)(piece - k.first[ti]) * GN_PIECE, n = k.t[ti].n;
        const int len = (int)(n - base < GN_PIECE ? n - base : GN_PIECE);
        if (k.dtype[ti] == RFX_F32) norm_piece<float, MAX>((const float*)k.t[ti].g + base, len, sum, big);
        else if (k.dtype[ti] == RFX_BF16) norm_piece<__bf16, MAX>((const __bf16*)k.t[ti].g + base, len, sum, big);
        else norm_piece<_Float16, MAX>((const _Float16*)k.t[ti].g + base, len, sum, big);
    }
    const double r = MAX ? block_max((double)__uint_as_float(big), lds) : block_sum(sum, lds);
    if (threadIdx.x == 0) k.partial[blockIdx.x] = r;
}

template <bool MAX>
__global__ __launch_bounds__(GN_THREADS) void grad_norm_join_kernel(const double* partial, int n, double max_norm, double* clip, float* norm32) {
    __shared__ double lds[GN_THREADS / 64];
    double x = 0.0;
    for (int i = threadIdx.x; i < n; i += GN_THREADS) {
        if (MAX) x = x != x ? x : (partial[i] != partial[i] || partial[i] > x) ? partial[i] : x;
        else x += partial[i];
    }
    x = MAX ? block_max(x, lds) : sqrt(block_sum(x, lds));
    if (threadIdx.x == 0) {
        const double f = max_norm / (x + 1e-6);
        clip[0] = x;
        clip[1] = f > 1.0 ? 1.0 : f;                                       // NaN stays NaN
        if (norm32) *norm32 = (float)x;
    }
}

template <typename T> __device__ __forceinline__ void scale_piece(T* g, int len, float c) {
    int done = 0;
    if (((uintptr_t)g & (4 * sizeof(T) - 1)) == 0) {
        done = len & ~3;
        for (int i = threadIdx.x * 4; i < done; i += GN_THREADS * 4) store4(g + i, load4(g + i) * c);
    }
    for (int i = done + threadIdx.x; i < len; i += GN_THREADS) g[i] = (T)((float)g[i] * c);
}

__global__ __launch_bounds__(GN_THREADS) void grad_scale_kernel(const GnArgs k) {
    const double f = k.clip[1];
    if (f == 1.0) return;
    const float c = (float)f;
    for (int piece = blockIdx.x; piece < k.pieces; piece += gridDim.x) {
        const int ti = find(k.first, k.count, piece);
        const int64_t base = (int64_t)(piece - k.first[ti]) * GN_PIECE, n = k.t[ti].n;
        const int len = (int)(n - base < GN_PIECE ? n - base : GN_PIECE);
        if (k.dtype[ti] == RFX_F32) scale_piece((float*)k.t[ti].g + base, len, c);
        else if (k.dtype[ti] == RFX_BF16) scale_piece((__bf16*)k.t[ti].g + base, len, c);
        else scale_piece((_Float16*)k.t[ti].g + base, len, c);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
static int elem_bytes(int dtype) { return dtype == RFX_F32 ? 4 : 2; }

// one launch of the tensors gathered in `k`; dev: their scalars' place in the workspace (step counts on the device)
static int adamw_launch(AwArgs& k, PrepArgs* prep, int kind, hipStream_t stream) {
    if (k.count == 0) return RFX_OK;
    if (prep) {
        prep->count = k.count;
        hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(64), 0, stream, *prep);
        RFX_LAUNCH_CHECK();
        k.dev = prep->out;
        prep->out += k.count;
    }
    if (k.first[k.count] == 0) {                                           // tensors without elements: their counts rise all the same
        k.count = 0;
        return RFX_OK;
    }
    const dim3 grid((unsigned)k.first[k.count]), block(AW_THREADS);
    switch (kind) {
        case 0: hipLaunchKernelGGL((adamw32_kernel<RFX_F32, false>), grid, block, 0, stream, k); break;
        case 1: hipLaunchKernelGGL((adamw32_kernel<RFX_BF16, false>), grid, block, 0, stream, k); break;
        case 2: hipLaunchKernelGGL((adamw32_kernel<RFX_F16, false>), grid, block, 0, stream, k); break;
        case 4: hipLaunchKernelGGL((adamw32_kernel<RFX_BF16, true>), grid, block, 0, stream, k); break;
        case 5: hipLaunchKernelGGL((adamw32_kernel<RFX_F16, true>), grid, block, 0, stream, k); break;
        case 6: hipLaunchKernelGGL((adamw8_kernel<RFX_F32, false>), grid, block, 0, stream, k); break;
        case 7: hipLaunchKernelGGL((adamw8_kernel<RFX_BF16, false>), grid, block, 0, stream, k); break;
        case 8: hipLaunchKernelGGL((adamw8_kernel<RFX_F16, false>), grid, block, 0, stream, k); break;
        case 10: hipLaunchKernelGGL((adamw8_kernel<RFX_BF16, true>), grid, block, 0, stream, k); break;
        case 11: hipLaunchKernelGGL((adamw8_kernel<RFX_F16, true>), grid, block, 0, stream, k); break;
        default: return RFX_ERR_ARG;
    }
    RFX_LAUNCH_CHECK();
    k.count = 0;
    return RFX_OK;
}

static int kind_of(const rfx_adamw_tensor& t, const rfx_adamw_group& g) { return t.dtype + (t.master ? 3 : 0) + (g.state_bits == 8 ? 6 : 0); }

static bool tensor_ok(const rfx_adamw_tensor& t, const rfx_adamw_group* groups, int n_groups) {
    if (t.n < 0 || t.group < 0 || t.group >= n_groups || t.dtype < RFX_F32 || t.dtype > RFX_F16) return false;
    const rfx_adamw_group& g = groups[t.group];
    if (!t.step_dev && (g.step < 1 || g.lr_dev)) return false;
    if (t.master && t.dtype == RFX_F32) return false;
    if (t.n == 0) return true;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return false;
    const uintptr_t low = elem_bytes(t.dtype) - 1;
    if (((uintptr_t)t.param | (uintptr_t)t.grad) & low) return false;
    if (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq | (uintptr_t)t.master | (uintptr_t)t.step_dev) & 3) return false;
    return g.state_bits != 8 || t.exponents;
}

static bool group_ok(const rfx_adamw_group& g) {
    return (g.state_bits == 32 || g.state_bits == 8) && g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0;
}

static bool overlap(const rfx_adamw_tensor& a, const rfx_adamw_tensor& b) {
    const uintptr_t a0 = (uintptr_t)a.param, b0 = (uintptr_t)b.param;
    return a0 < b0 + (uintptr_t)b.n * elem_bytes(b.dtype) && b0 < a0 + (uintptr_t)a.n * elem_bytes(a.dtype);
}

// pieces of the gradients [at, at + as many as fit) as one launch; returns how many were taken, 0: none left, < 0: an error.
// apart: no two of a launch share memory (they are written)
static int gather(const rfx_grad_tensor* t, int count, int& at, GnArgs& k, bool apart) {
    int64_t pieces = 0;
    k.count = 0;
    for (; at < count && k.count < GN_TENSORS; ++at) {
        if (t[at].n == 0) continue;
        bool shared = false;
        for (int j = 0; apart && !shared && j < k.count; ++j) {
            const uintptr_t a = (uintptr_t)t[at].grad, b = (uintptr_t)k.t[j].g;
            shared = a < b + (uintptr_t)k.t[j].n * elem_bytes(k.dtype[j]) && b < a + (uintptr_t)t[at].n * elem_bytes(t[at].dtype);
        }
        if (shared) break;
        const int64_t p = (t[at].n + GN_PIECE - 1) / GN_PIECE;
        if (p > 0x7fffffff) return RFX_ERR_UNSUPPORTED;
        if (pieces + p > 0x7fffffff) break;
        k.t[k.count].g = t[at].grad;
        k.t[k.count].n = t[at].n;
        k.dtype[k.count] = (uint8_t)t[at].dtype;
        k.first[k.count++] = (int32_t)pieces;
        pieces += p;
    }
    k.first[k.count] = k.pieces = (int32_t)pieces;
    return k.count;
}

static bool grads_ok(const rfx_grad_tensor* t, int count) {
    if (count < 0 || (count > 0 && !t)) return false;
    for (int i = 0; i < count; ++i) {
        if (t[i].n < 0 || t[i].dtype < RFX_F32 || t[i].dtype > RFX_F16) return false;
        if (t[i].n > 0 && (!t[i].grad || ((uintptr_t)t[i].grad & (uintptr_t)(elem_bytes(t[i].dtype) - 1)))) return false;
    }
    return true;
}

static int norm_blocks(int pieces) { return pieces < GN_BLOCKS ? pieces : GN_BLOCKS; }

}  // namespace rfx

using namespace rfx;

extern "C" {

size_t rfx_adamw_tensor_bytes(void) { return sizeof(rfx_adamw_tensor); }
size_t rfx_adamw_group_bytes(void) { return sizeof(rfx_adamw_group); }
size_t rfx_adamw_workspace_bytes(int count) { return count > 0 ? (size_t)count * sizeof(AwStep) : 0; }

int rfx_adamw_step(const rfx_adamw_tensor* tensors, int count, const rfx_adamw_group* groups, int n_groups, const double* clip,
                   void* workspace, size_t workspace_bytes, rfx_stream stream) {
    if (count == 0) return RFX_OK;
    if (!tensors || count < 0 || !groups || n_groups < 1) return RFX_ERR_ARG;
    bool on_device = false;
    unsigned kinds = 0;
    for (int i = 0; i < n_groups; ++i)
        if (!group_ok(groups[i])) return RFX_ERR_ARG;
    for (int i = 0; i < count; ++i) {
        if (!tensor_ok(tensors[i], groups, n_groups)) return RFX_ERR_ARG;
        if ((tensors[i].n + AW_PIECE - 1) / AW_PIECE > 0x7fffffff) return RFX_ERR_UNSUPPORTED;
        on_device |= tensors[i].step_dev != nullptr;
        kinds |= 1U << kind_of(tensors[i], groups[tensors[i].group]);
    }
    if (on_device && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < rfx_adamw_workspace_bytes(count))) return RFX_ERR_WORKSPACE;
    AwArgs k;
    PrepArgs prep;
    prep.out = (AwStep*)workspace;
    k.clip = clip;
    for (int kind = 0; kind < 12; ++kind) {
        if (!(kinds >> kind & 1)) continue;
        for (int counted = 0; counted < 2; ++counted) {                    // step counts from the host, then those on the device
            if (counted && !on_device) break;
            int at[AW_TENSORS], group_at[AW_GROUPS], used = 0;
            int64_t blocks = 0;
            k.count = 0;
            k.dev = nullptr;
            for (int i = 0; i <= count; ++i) {
                if (i < count) {
                    const rfx_adamw_tensor& t = tensors[i];
                    if (kind_of(t, groups[t.group]) != kind || (t.step_dev != nullptr) != (counted != 0)) continue;
                    if (t.n == 0 && !counted) continue;
                    const int64_t pieces = (t.n + AW_PIECE - 1) / AW_PIECE;
                    int gi = 0;
                    while (gi < used && group_at[gi] != t.group) ++gi;
                    bool full = k.count == AW_TENSORS || gi == AW_GROUPS || blocks + pieces > 0x7fffffff;
                    for (int j = 0; !full && j < k.count; ++j) full = overlap(t, tensors[at[j]]);
                    if (!full) {
                        if (gi == used) {
                            const rfx_adamw_group& g = groups[t.group];
                            AwGroup& a = k.group[gi];
                            a.b1 = g.beta1; a.c1 = 1.0 - g.beta1; a.b2 = g.beta2; a.c2 = 1.0 - g.beta2;
                            a.eps = (float)g.eps;
                            a.sign = g.maximize ? -1.f : 1.f;
                            if (!counted) a.s = step_scalars(g.lr, g.beta1, g.beta2, g.weight_decay, (double)g.step, g.seed);
                            prep.g[gi] = {g.lr, g.beta1, g.beta2, g.weight_decay, g.lr_dev, g.seed};
                            group_at[used++] = t.group;
                        }
                        at[k.count] = i;
                        k.t[k.count] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exponents, t.master, t.n, gi, t.index};
                        prep.step[k.count] = t.step_dev;
                        prep.group[k.count] = (uint8_t)gi;
                        k.first[k.count++] = (int32_t)blocks;
                        blocks += pieces;
                        k.first[k.count] = (int32_t)blocks;
                        continue;
                    }
                    --i;                                                   // again, as the first of the next launch
                }
                const int rc = adamw_launch(k, counted ? &prep : nullptr, kind, as_stream(stream));
                if (rc != RFX_OK) return rc;
                used = 0;
                blocks = 0;
            }
        }
    }
    return RFX_OK;
}

int rfx_adamw_moments(const rfx_moment_tensor* tensors, int count, rfx_stream stream) {
    if (count == 0) return RFX_OK;
    if (!tensors || count < 0) return RFX_ERR_ARG;
    for (int i = 0; i < count; ++i) {
        const rfx_moment_tensor& t = tensors[i];
        if (t.n < 0 || (t.n > 0 && (!t.exp_avg || !t.exp_avg_sq || !t.exponents || !t.out_avg || !t.out_avg_sq))) return RFX_ERR_ARG;
        if (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq | (uintptr_t)t.out_avg | (uintptr_t)t.out_avg_sq) & 3) return RFX_ERR_ARG;
        if ((t.n + AW_PIECE - 1) / AW_PIECE > 0x7fffffff) return RFX_ERR_UNSUPPORTED;
    }
    MomArgs k;
    for (int i = 0; i < count;) {
        int64_t blocks = 0;
        for (k.count = 0; i < count && k.count < AW_TENSORS; ++i) {
            if (tensors[i].n == 0) continue;
            const int64_t pieces = (tensors[i].n + AW_PIECE - 1) / AW_PIECE;
            if (blocks + pieces > 0x7fffffff) break;
            k.t[k.count] = tensors[i];
            k.first[k.count++] = (int32_t)blocks;
            blocks += pieces;
        }
        if (k.count == 0) break;
        k.first[k.count] = (int32_t)blocks;
        hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)blocks), dim3(AW_THREADS), 0, as_stream(stream), k);
        RFX_LAUNCH_CHECK();
    }
    return RFX_OK;
}

size_t rfx_grad_norm_workspace_bytes(const rfx_grad_tensor* tensors, int count) {
    if (!grads_ok(tensors, count)) return 0;
    size_t n = 0;
    GnArgs k;
    for (int at = 0; gather(tensors, count, at, k, false) > 0;) n += norm_blocks(k.pieces);
    return (n ? n : 1) * sizeof(double);
}

int rfx_grad_norm(const rfx_grad_tensor* tensors, int count, int norm_type, double max_norm, double* clip, float* norm32,
                  void* workspace, size_t workspace_bytes, rfx_stream stream) {
    if (!grads_ok(tensors, count) || !clip || ((uintptr_t)clip & 7) || !(max_norm >= 0.0)) return RFX_ERR_ARG;
    if (norm_type != 2 && norm_type != 0) return RFX_ERR_UNSUPPORTED;
    if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < rfx_grad_norm_workspace_bytes(tensors, count)) return RFX_ERR_WORKSPACE;
    GnArgs k;
    double* partial = (double*)workspace;
    int n = 0;
    for (int at = 0;;) {
        const int taken = gather(tensors, count, at, k, false);
        if (taken < 0) return taken;
        if (taken == 0) break;
        const int blocks = norm_blocks(k.pieces);
        k.partial = partial + n;
        n += blocks;
        if (norm_type == 2) hipLaunchKernelGGL(grad_norm_kernel<false>, dim3(blocks), dim3(GN_THREADS), 0, as_stream(stream), k);
        else hipLaunchKernelGGL(grad_norm_kernel<true>, dim3(blocks), dim3(GN_THREADS), 0, as_stream(stream), k);
        RFX_LAUNCH_CHECK();
    }
    if (norm_type == 2) hipLaunchKernelGGL(grad_norm_join_kernel<false>, dim3(1), dim3(GN_THREADS), 0, as_stream(stream), partial, n, max_norm, clip, norm32);
    else hipLaunchKernelGGL(grad_norm_join_kernel<true>, dim3(1), dim3(GN_THREADS), 0, as_stream(stream), partial, n, max_norm, clip, norm32);
    RFX_LAUNCH_CHECK();
    return RFX_OK;
}

int rfx_grad_clip(const rfx_grad_tensor* tensors, int count, int norm_type, double max_norm, double* clip, float* norm32,
                  void* workspace, size_t workspace_bytes, rfx_stream stream) {
    const int rc = rfx_grad_norm(tensors, count, norm_type, max_norm, clip, norm32, workspace, workspace_bytes, stream);
    return rc == RFX_OK ? rfx_grad_scale(tensors, count, clip, stream) : rc;
}

int rfx_grad_scale(const rfx_grad_tensor* tensors, int count, const double* clip, rfx_stream stream) {
    if (!grads_ok(tensors, count) || !clip) return RFX_ERR_ARG;
    GnArgs k;
    k.clip = clip;
    for (int at = 0;;) {
        const int taken = gather(tensors, count, at, k, true);
        if (taken < 0) return taken;
        if (taken == 0) break;
        hipLaunchKernelGGL(grad_scale_kernel, dim3(k.pieces), dim3(GN_THREADS), 0, as_stream(stream), k);
        RFX_LAUNCH_CHECK();
    }
    return RFX_OK;
}

}  // extern "C"
