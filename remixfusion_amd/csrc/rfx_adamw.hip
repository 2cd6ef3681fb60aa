// rfx_adamw.hip -- AdamW over many tensors (moments in 32 or in 8 bits), the gradients' global norm and their scaling.
//
// Every kernel here is one pass over its data: an element of the step costs 28 bytes (fp32 parameter, 32-bit moments) or 16
// (8-bit moments) of HBM traffic and some dozens of vector instructions, so the bytes are the bound and the instructions are
// what has to stay under them.  All tensors of a kind (type, state, master copy) go into one launch: their descriptors travel in
// the kernel's arguments (no table in device memory that a later call could overwrite under a running kernel or a captured one),
// every tensor is cut into pieces of AW_PIECE elements, and a block finds its tensor by bisection over the first pieces.
#include "rfx_common.h"
#include <math.h>

namespace rfx {

constexpr int AW_THREADS = 256;
// Elements per block: four a thread, one run of the 8-bit form a wave.  Small blocks fill the chip early and leave no tail: 135 000 parameters
// in 8 bits step in 4.6 us, with 4096 elements a block in 6.3; 41.5 million in 32 bits in 189 us, with 4096 in 205.
constexpr int AW_PIECE = AW_THREADS * 4;
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
    int32_t wide;                       // 8 bits: byte of a run's second moments from which its update is formed in fp64
};

// Runs of 8-bit moments whose denominators fp32 does not hold.  Scaled by the run's largest (2^e), a root of v under 2^(e - 113) is not normal
// there: it may be lost next to an eps that is 2^35 times as large (ten bits of it for 1 / sqrt(1 - b2^k)), else m / eps would be a leap.  And
// the chip's reciprocal makes 0 of what would be under 2^-126: roots from 2^91 on, with room for the same ten bits and for lr m.  A run is wide
// from roots of 2^28 on with eps = 1e-15, of 2^51 with 1e-8; all others pay a comparison of scalars (41.6 million parameters 162 us as before).
static int wide_from(double eps) {
    const int e = eps > 0.0 && eps < 0x1p100 ? ilogb(eps) + 113 - 35 : -128;
    return e < -128 ? -128 : e < 91 ? e : 91;
}

// Where the clipping factor comes from: partial sums (maxima) of the norm that every wave joins for itself -- never more than four a
// lane, out of L2, for a launch less -- or a factor that is there.  Neither: no clipping.
constexpr int JOIN = 256;
struct ClipSource {
    const double* partial;
    const double* factor;
    double max_norm;
    float* norm32;                      // written by the first block
    int32_t n;
    int32_t max;                        // maxima instead of sums of squares
};

struct AwArgs {
    AwTensor t[AW_TENSORS];
    int32_t first[AW_TENSORS + 1];
    AwGroup group[AW_GROUPS];
    const AwStep* dev;                  // per tensor of this launch, or null
    ClipSource clip;
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

// STREAM: past the caches, for sets that no cache holds until they are read again
template <bool STREAM = false, typename T> __device__ __forceinline__ f4 load4(const T* p) {
    const vec4<T>* at = reinterpret_cast<const vec4<T>*>(p);
    return widen(STREAM ? __builtin_nontemporal_load(at) : *at);
}
template <bool STREAM = false, typename T> __device__ __forceinline__ void store4(T* p, f4 x) {
    vec4<T> y;
    if constexpr (sizeof(T) == 4) y = x;
    else y = __builtin_convertvector(x, vec4<T>);                          // to nearest, ties to even: once, at the end
    vec4<T>* at = reinterpret_cast<vec4<T>*>(p);
    if (STREAM) __builtin_nontemporal_store(y, at); else *at = y;
}

// xor-shift / multiply mixer of 32-bit integers (a bijection): shifts and multipliers as published by C. Wellons in 2018, the least biased of
// the two-multiply mixers that he searched
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

// p - (lr wd p + update): the two small terms meet before they meet p, so a decay of less than half a unit of p's last place is not
// lost to a rounding of its own.  An infinite p stays what p (1 - lr wd) leaves it
__device__ __forceinline__ float stepped(float p, float update, float lr_wd) {
    return p - (fabsf(p) == __builtin_inff() ? update : madd(lr_wd, p, update));
}

// A clipping factor as fp32 products take it: norms beyond 2^100 limits would make one that is subnormal there, or nothing
struct Factor32 {
    float f, unit;
    __device__ explicit Factor32(double x) : f((float)(x < 0x1p-100 ? x * 0x1p100 : x)), unit(x < 0x1p-100 ? 0x1p-100f : 1.f) {}
};

// ---- 32-bit moments: fp32 throughout ------------------------------------------------------------------------------------------
// Bound by HBM: 28 bytes an fp32 element, 41.5 million in 189 us = 6.1 TB/s (a large copy: 5.4).
__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, const AwGroup& a, const AwStep& s, Factor32 c) {
    const float c1 = (float)a.c1, c2 = (float)a.c2, b1 = (float)a.b1, b2 = (float)a.b2;
    g = g * c.f * c.unit;
    m = madd(c1, g, b1 * m);
    v = madd(c2 * g, g, b2 * v);
    p = stepped(p, s.step_size * (m / madd(sqrtf(v), s.inv_bc2, a.eps)), s.lr_wd);
}

__device__ __forceinline__ double larger(double p, double q) { return p != p ? p : (q != q || q > p) ? q : p; }     // NaN wins

template <int THREADS> __device__ __forceinline__ double block_join(double x, bool max, double* lds) {      // every thread gets it; fixed order
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const double y = __shfl_xor(x, d, 64);
        x = max ? larger(x, y) : x + y;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) x = max ? larger(x, lds[w]) : x + lds[w];
    return x;
}

__device__ __forceinline__ double factor_of(double norm, double max_norm) {
    const double f = max_norm / (norm + 1e-6);
    return f > 1.0 ? 1.0 : f;                                              // NaN stays NaN
}

// each wave for itself, so that nothing waits at a barrier
__device__ __forceinline__ double clip_factor(const ClipSource& c) {
    if (c.n == 0) return c.factor ? c.factor[1] : 1.0;
    double x = 0.0;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < JOIN; i += 64) {
        const double y = i + lane < c.n ? c.partial[i + lane] : 0.0;
        x = c.max ? larger(x, y) : x + y;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const double y = __shfl_xor(x, d, 64);
        x = c.max ? larger(x, y) : x + y;
    }
    const double norm = c.max ? x : sqrt(x);
    if (c.norm32 && blockIdx.x == 0 && threadIdx.x == 0) *c.norm32 = (float)norm;
    return factor_of(norm, c.max_norm);
}

template <int TYPE, bool MASTER, bool STREAM>
__global__ __launch_bounds__(AW_THREADS) void adamw32_kernel(const AwArgs k) {
    typedef typename Elem<TYPE>::T T;
    const int ti = find(k.first, k.count, (int)blockIdx.x);
    const AwTensor& t = k.t[ti];
    const AwGroup& a = k.group[t.group];
    const AwStep s = k.dev ? k.dev[ti] : a.s;
    Factor32 c(clip_factor(k.clip));
    c.f *= a.sign;
    const int64_t base = (int64_t)((int)blockIdx.x - k.first[ti]) * AW_PIECE;
    const int len = (int)(t.n - base < AW_PIECE ? t.n - base : AW_PIECE);
    T* p = (T*)t.p + base;
    const T* g = (const T*)t.g + base;
    float* m = (float*)t.m + base;
    float* v = (float*)t.v + base;
    float* w = MASTER ? t.w + base : nullptr;
    const bool vec = ((((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) | (((uintptr_t)m | (uintptr_t)v | (uintptr_t)w) & 15)) == 0;
    int i = threadIdx.x * 4;
    if (vec && i + 4 <= len) {
        f4 x = MASTER ? load4<STREAM>(w + i) : load4<STREAM>(p + i);
        const f4 gg = load4<STREAM>(g + i);
        f4 mm = load4<STREAM>(m + i), vv = load4<STREAM>(v + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float xj = x[j], mj = mm[j], vj = vv[j];
            adamw_one(xj, gg[j], mj, vj, a, s, c);
            x[j] = xj; mm[j] = mj; vv[j] = vj;
        }
        store4<STREAM>(p + i, x);
        if (MASTER) store4<STREAM>(w + i, x);
        store4<STREAM>(m + i, mm);
        store4<STREAM>(v + i, vv);
        return;
    }
    int step = 1, end = i + 4 < len ? i + 4 : len;                         // the last elements of a tensor: those of this lane
    if (!vec) { i = threadIdx.x; step = AW_THREADS; end = len; }           // no vector load fits: neighbours to neighbouring lanes
    for (; i < end; i += step) {
        float x = MASTER ? w[i] : (float)p[i], mm = m[i], vv = v[i];
        adamw_one(x, (float)g[i], mm, vv, a, s, c);
        p[i] = (T)x;
        if (MASTER) w[i] = x;
        m[i] = mm; v[i] = vv;
    }
}

// ---- 8-bit moments ------------------------------------------------------------------------------------------------------------
// A wave owns a run of 256 elements, four consecutive ones a lane.  The moments are formed in fp64 (full rate on this chip), so
// that which side of a border they fall on does not depend on the order of the operations; the update is fp32 (of wide runs fp64).
//   decode: a byte's seven (eight) bits moved to an fp32's exponent and mantissa ARE the format, subnormals included, times a power
//           of two that is a constant of the run (beta goes into it: a product with a power of two is exact);
//   encode: the moment times the inverse power of two, rounded to fp32 (subnormals included), leaves 20 bits below the format's
//           last place: 16 random bits (and half of their unit) are added, and the upper bits are the code.
// Why at random: one step moves an average by (1 - beta) of its distance -- a thousandth for beta2 = 0.999 -- and the formats' places
// are an eighth apart; to nearest, the average would stand still.  Why second moments never become 0: m / eps would be a leap.
// 16 bytes an fp32 element and 76 vector instructions: 41.5 million in 105-111 us = 6.0-6.3 TB/s, of them 80 us of instructions (4.9e7 a
// launch over 1024 SIMDs at four cycles each).  3 million fp16 parameters, 30 MB that the caches hold: 12 us, of them 6 of instructions and
// the rest the launch's own rise and fall (a CU is busy for 8.6).  The codes are read and written through the
// caches also where the rest goes past them: four bytes a lane, they share their lines with other waves.
__device__ __forceinline__ double pow2(int e) { return __longlong_as_double((long long)(e + 1023) << 52); }

template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);       // lanes without a source: 0
    return x > y ? x : y;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {                 // a scalar
    x = dpp_max<0x111, 0xf>(x);                                            // from the lane 1, 2, 4, 8 to the left in a row of 16
    x = dpp_max<0x112, 0xf>(x);
    x = dpp_max<0x114, 0xf>(x);
    x = dpp_max<0x118, 0xf>(x);
    x = dpp_max<0x142, 0xa>(x);                                            // a row's last lane to the next row
    x = dpp_max<0x143, 0xc>(x);                                            // lane 31 to the upper half
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
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

template <int J> __device__ __forceinline__ float bits_m(uint32_t codes) {
    const uint32_t x = codes << (24 - 8 * J);
    return __uint_as_float((x & 0x80000000U) | ((x >> 4) & 0x07f00000U));
}
template <int J> __device__ __forceinline__ float bits_v(uint32_t codes) {
    return __uint_as_float((J < 3 ? codes << (24 - 8 * J) : codes) >> 4 & 0x0ff00000U);
}

template <uint32_t TOP> __device__ __forceinline__ uint32_t encode(double magnitude, double inverse, uint32_t noise) {
    const uint32_t c = (__float_as_uint((float)(magnitude * inverse)) + noise) >> 20;
    return c < TOP ? c : TOP;
}

struct Run8 {                           // a lane's share of a run as it is loaded
    f4 x, g;
    uint32_t cm, cv;
    int e1, e2;
};

// new moments of a lane's elements (codes in r.cm, r.cv), the stepped parameter in r.x, the run's exponents in r.e1, r.e2
template <bool FULL> __device__ __forceinline__ void adamw8_run(Run8& r, const AwGroup& a, const AwStep& s, double c, uint32_t run_key, int lane, int have) {
    const double s1 = scale_m(__builtin_amdgcn_readfirstlane(r.e1)) * a.b1, s2 = scale_v(__builtin_amdgcn_readfirstlane(r.e2)) * a.b2;
    const float bm[4] = {bits_m<0>(r.cm), bits_m<1>(r.cm), bits_m<2>(r.cm), bits_m<3>(r.cm)};
    const float bv[4] = {bits_v<0>(r.cv), bits_v<1>(r.cv), bits_v<2>(r.cv), bits_v<3>(r.cv)};
    double m[4], v[4];
    uint32_t h1 = 0, h2 = 0, u2[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double g = (double)r.g[j] * c;
        m[j] = fma(g, a.c1, (double)bm[j] * s1);
        v[j] = fma(g * g, a.c2, (double)bv[j] * s2);
        const uint32_t u1 = (uint32_t)__double2hiint(m[j]) & 0x7fffffffU;
        u2[j] = (uint32_t)__double2hiint(v[j]) & 0x7fffffffU;
        if (FULL || j < have) { h1 = h1 > u1 ? h1 : u1; h2 = h2 > u2[j] ? h2 : u2[j]; }
    }
    r.e1 = run_exponent<1>(wave_max(h1));
    r.e2 = run_exponent<2>(wave_max(h2));
    const double i1 = pow2(-112 - r.e1), i2 = pow2(-96 - 2 * r.e2);
    // the root is taken of v 2^(2 half), which no fp32 overflows; what underflows there is nothing next to eps, or the run is wide
    const int half = r.e2 < -50 ? 100 : 50 - r.e2;
    const double up = pow2(2 * half);
    const float down = s.inv_bc2 * __uint_as_float((uint32_t)(127 - half) << 23);
    const bool wide = r.e2 == -128 || r.e2 >= a.wide;                      // (a scalar)
    r.cm = r.cv = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t bits = mix32(run_key + (uint32_t)(lane * 4 + j) * 0x9e3779b9U);
        // 16 bits at the place 2^4 of the 20, and half of a unit of theirs
        const uint32_t cm = encode<127>(fabs(m[j]), i1, ((bits & 0xffffU) << 4) | 8U);
        uint32_t cv = encode<255>(v[j], i2, (bits >> 16 << 4) | 8U);
        const uint32_t some = u2[j] < 1U ? u2[j] : 1U;                     // v > 0 stays above 0: m / eps would be a leap
        cv = cv > some ? cv : some;
        r.cm |= (cm | ((uint32_t)__double2hiint(m[j]) >> 24 & 128U)) << (8 * j);
        r.cv |= cv << (8 * j);
        float update;
        if (wide) {
            update = (float)((double)s.step_size * m[j] / (sqrt(v[j]) * s.inv_bc2 + a.eps));
        } else {                                                           // fp32, the chip's own root and reciprocal: an ulp each, under 16 u all told
            const float d = madd(__builtin_amdgcn_sqrtf((float)(v[j] * up)), down, a.eps);
            update = s.step_size * (float)m[j] * __builtin_amdgcn_rcpf(d);
        }
        r.x[j] = stepped(r.x[j], update, s.lr_wd);
    }
}

template <int TYPE, bool MASTER, bool STREAM>
__global__ __launch_bounds__(AW_THREADS) void adamw8_kernel(const AwArgs k) {
    typedef typename Elem<TYPE>::T T;
    const int ti = find(k.first, k.count, (int)blockIdx.x);
    const AwTensor& t = k.t[ti];
    const AwGroup& a = k.group[t.group];
    const AwStep s = k.dev ? k.dev[ti] : a.s;
    const double c = (double)a.sign * clip_factor(k.clip);
    const int64_t piece = (int)blockIdx.x - k.first[ti];
    const int64_t base = piece * AW_PIECE;
    const int len = (int)(t.n - base < AW_PIECE ? t.n - base : AW_PIECE);
    const int64_t runs = (t.n + AW_RUN - 1) / AW_RUN, run0 = piece * (AW_PIECE / AW_RUN);
    const uint32_t key = mix32(s.key + t.index) + (uint32_t)run0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T* g = (const T*)t.g + base;
    T* p = (T*)t.p + base;
    float* w = MASTER ? t.w + base : nullptr;
    uint8_t* m = (uint8_t*)t.m + base;
    uint8_t* v = (uint8_t*)t.v + base;
    int8_t* e1 = t.e + run0;
    int8_t* e2 = t.e + runs + run0;
    const bool vec = ((((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) | ((uintptr_t)w & 15)) == 0;
    const int run = wave, i = run * AW_RUN + lane * 4;
    const uint32_t run_key = mix32(key + (uint32_t)run);
    Run8 x;
    if (len == AW_PIECE && vec) {
        x.x = MASTER ? load4<STREAM>(w + i) : load4<STREAM>(p + i);
        x.g = load4<STREAM>(g + i);
        x.cm = *reinterpret_cast<const uint32_t*>(m + i);
        x.cv = *reinterpret_cast<const uint32_t*>(v + i);
        x.e1 = e1[run];
        x.e2 = e2[run];
        adamw8_run<true>(x, a, s, c, run_key, lane, 4);
        store4<STREAM>(p + i, x.x);
        if (MASTER) store4<STREAM>(w + i, x.x);
        *reinterpret_cast<uint32_t*>(m + i) = x.cm;
        *reinterpret_cast<uint32_t*>(v + i) = x.cv;
    } else {                                                               // a tensor's last piece, or one that vector loads do not fit
        if (run * AW_RUN >= len) return;
        const int have = len - i < 0 ? 0 : len - i > 4 ? 4 : len - i;      // elements of this lane
        x = Run8{};
        for (int j = 0; j < have; ++j) {
            x.x[j] = MASTER ? w[i + j] : (float)p[i + j];
            x.g[j] = (float)g[i + j];
            x.cm |= (uint32_t)m[i + j] << (8 * j);
            x.cv |= (uint32_t)v[i + j] << (8 * j);
        }
        x.e1 = e1[run];
        x.e2 = e2[run];
        adamw8_run<false>(x, a, s, c, run_key, lane, have);
        for (int j = 0; j < have; ++j) {
            p[i + j] = (T)x.x[j];
            if (MASTER) w[i + j] = x.x[j];
            m[i + j] = (uint8_t)(x.cm >> (8 * j));
            v[i + j] = (uint8_t)(x.cv >> (8 * j));
        }
    }
    if (lane == 0) { e1[run] = (int8_t)x.e1; e2[run] = (int8_t)x.e2; }
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

template <bool STREAM>
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
    const int i = threadIdx.x * 4;
    if (i < len) {
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
        const auto value = [](float bits, double scale) { return (float)((double)bits * scale); };
        const f4 a = {value(bits_m<0>(cm), s1), value(bits_m<1>(cm), s1), value(bits_m<2>(cm), s1), value(bits_m<3>(cm), s1)};
        const f4 b = {value(bits_v<0>(cv), s2), value(bits_v<1>(cv), s2), value(bits_v<2>(cv), s2), value(bits_v<3>(cv), s2)};
        if (have == 4 && vec) {
            store4<STREAM>(om + i, a);
            store4<STREAM>(ov + i, b);
        } else {
            for (int j = 0; j < have; ++j) { om[i + j] = a[j]; ov[i + j] = b[j]; }
        }
    }
}

// ---- global norm --------------------------------------------------------------------------------------------------------------
// One block per CU at most (16 waves, four loads of each in flight: enough to draw what HBM gives), so that there are never more
// partial results than the blocks that read them join with one load a thread.  Each block has one piece, in whole rounds of its four
// loads: 166 MB in 30 us (5.5 TB/s, what a large copy reaches); eight smaller pieces a block, dealt in turn, cost 2 us more, eight loads in
// flight 6.  fp64 sums: no square of an fp32 number overflows or vanishes there, and the order -- pieces, lanes, waves, blocks -- is
// fixed by the sizes alone.
constexpr int GN_TENSORS = 128;
constexpr int GN_THREADS = 1024;
constexpr int64_t GN_ROUND = 4 * GN_THREADS;       // elements: one float4 a thread

struct GnArgs {
    struct { void* g; int64_t n; } t[GN_TENSORS];
    int32_t first[GN_TENSORS + 1];
    uint8_t dtype[GN_TENSORS];
    double* partial;
    ClipSource clip;
    int32_t count, pieces, piece, max;
};
static_assert(sizeof(GnArgs) <= 4096, "kernel arguments");

// a lane's four neighbours wherever they start: the sums' order must not depend on an address
template <typename T> __device__ __forceinline__ f4 load4_at(const T* p) {
    typedef T any4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    return widen((vec4<T>)*reinterpret_cast<const any4*>(p));
}

template <typename T, bool MAX> __device__ __forceinline__ void norm_piece(const T* g, int len, double& sum, uint32_t& big) {
    const auto one = [&](float x) {
        if (MAX) { const uint32_t u = __float_as_uint(x) & 0x7fffffffU; big = big > u ? big : u; }      // integers order NaN above all
        else { const double d = (double)x; sum = fma(d, d, sum); }
    };
    const auto four = [&](f4 x) {
#pragma unroll
        for (int j = 0; j < 4; ++j) one(x[j]);
    };
    const int done = len & ~3;
    int i = threadIdx.x * 4;
    for (; i + 3 * GN_THREADS * 4 < done; i += 4 * GN_THREADS * 4) {
        const f4 a = load4_at(g + i), b = load4_at(g + i + GN_THREADS * 4), c = load4_at(g + i + 2 * GN_THREADS * 4), d = load4_at(g + i + 3 * GN_THREADS * 4);
        four(a); four(b); four(c); four(d);
    }
    for (; i < done; i += GN_THREADS * 4) four(load4_at(g + i));
    for (i = done + threadIdx.x; i < len; i += GN_THREADS) one((float)g[i]);
}

template <bool MAX>
__global__ __launch_bounds__(GN_THREADS) void grad_norm_kernel(const GnArgs k) {
    __shared__ double lds[GN_THREADS / 64];
    double sum = 0.0;
    uint32_t big = 0;
    for (int piece = blockIdx.x; piece < k.pieces; piece += gridDim.x) {
        const int ti = find(k.first, k.count, piece);
        const int64_t base = (int64_t)(piece - k.first[ti]) * k.piece, n = k.t[ti].n;
        const int len = (int)(n - base < k.piece ? n - base : k.piece);
        if (k.dtype[ti] == RFX_F32) norm_piece<float, MAX>((const float*)k.t[ti].g + base, len, sum, big);
        else if (k.dtype[ti] == RFX_BF16) norm_piece<__bf16, MAX>((const __bf16*)k.t[ti].g + base, len, sum, big);
        else norm_piece<_Float16, MAX>((const _Float16*)k.t[ti].g + base, len, sum, big);
    }
    const double r = block_join<GN_THREADS>(MAX ? (double)__uint_as_float(big) : sum, MAX, lds);
    if (threadIdx.x == 0) k.partial[blockIdx.x] = r;
}

// partial results to the norm and its factor
__global__ __launch_bounds__(JOIN) void grad_norm_join_kernel(const double* partial, int n, int max, double max_norm, double* clip, float* norm32) {
    __shared__ double lds[JOIN / 64];
    double x = 0.0;
    for (int i = threadIdx.x; i < n; i += JOIN) x = max ? larger(x, partial[i]) : x + partial[i];
    x = block_join<JOIN>(x, max != 0, lds);
    if (threadIdx.x != 0) return;
    const double norm = max ? x : sqrt(x);
    if (clip) {
        clip[0] = norm;
        clip[1] = factor_of(norm, max_norm);
    }
    if (norm32) *norm32 = (float)norm;
}

// the norm's pieces on the blocks that the norm had them on: what an XCD's L2 still holds of a small set is found there (1.6 million
// gradients 5.8 us, in pieces of another size 7.4)
template <typename T> __device__ __forceinline__ void scale_piece(T* g, int len, Factor32 c) {
    int done = 0;
    if (((uintptr_t)g & (4 * sizeof(T) - 1)) == 0) {
        done = len & ~3;
        for (int i = threadIdx.x * 4; i < done; i += GN_THREADS * 4) store4(g + i, load4(g + i) * c.f * c.unit);
    }
    for (int i = done + threadIdx.x; i < len; i += GN_THREADS) g[i] = (T)((float)g[i] * c.f * c.unit);
}

__global__ __launch_bounds__(GN_THREADS) void grad_scale_kernel(const GnArgs k) {
    const double f = clip_factor(k.clip);
    if (f == 1.0) return;
    const Factor32 c(f);
    for (int piece = blockIdx.x; piece < k.pieces; piece += gridDim.x) {
        const int ti = find(k.first, k.count, piece);
        const int64_t base = (int64_t)(piece - k.first[ti]) * k.piece, n = k.t[ti].n;
        const int len = (int)(n - base < k.piece ? n - base : k.piece);
        if (k.dtype[ti] == RFX_F32) scale_piece((float*)k.t[ti].g + base, len, c);
        else if (k.dtype[ti] == RFX_BF16) scale_piece((__bf16*)k.t[ti].g + base, len, c);
        else scale_piece((_Float16*)k.t[ti].g + base, len, c);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
static int elem_bytes(int dtype) { return dtype == RFX_F32 ? 4 : 2; }

// From this much memory on (parameters, gradients, moments) the step's loads and stores go past the caches.
// Measured, us a step (plain loads and stores / past the caches), sets of fp32 tensors stepped again and again: 26 MB 9.6 / 11.0, 64 MB
// 19 / 22, 128 MB 43 / 39, 664 MB 217 / 191; behind other work on 256 MB, as in a training loop: 16 MB 13.6 / 7.6, 64 MB 37 / 22, 128 MB
// 64 / 40.  What is stepped next to nothing else stays in the caches under this size, and the larger sets gain either way.
// In the mapper, whose smallest table is 26 MB by this count, behind a render and its backward: 8.6 us plain and 9.9 past the caches in 32
// bits, 8.9 and 8.5 in 8; whole runs 2 109 and 2 082 frames/s in 32 bits, 2 086 and 2 083 in 8: under the size, plain.
constexpr int64_t STREAM_BYTES = 64 << 20;
static int64_t pieces_of(int64_t n) { return (n + AW_PIECE - 1) / AW_PIECE; }
constexpr int64_t AW_BLOCKS = 0xffffffffLL / AW_THREADS;                   // of a launch: its threads are counted in 32 bits
constexpr int64_t MOST_ELEMENTS = (int64_t)1 << 52;                        // sizes add up without overflow

// one launch of the tensors gathered in `k`; dev: their scalars' place in the workspace (step counts on the device)
static int adamw_launch(AwArgs& k, PrepArgs* prep, int kind, bool past, hipStream_t stream) {
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
    const void* kernel = nullptr;
    const auto pick = [&](auto plain, auto streaming) { kernel = past ? (const void*)streaming : (const void*)plain; };
    switch (kind) {
        case 0: pick(adamw32_kernel<RFX_F32, false, false>, adamw32_kernel<RFX_F32, false, true>); break;
        case 1: pick(adamw32_kernel<RFX_BF16, false, false>, adamw32_kernel<RFX_BF16, false, true>); break;
        case 2: pick(adamw32_kernel<RFX_F16, false, false>, adamw32_kernel<RFX_F16, false, true>); break;
        case 4: pick(adamw32_kernel<RFX_BF16, true, false>, adamw32_kernel<RFX_BF16, true, true>); break;
        case 5: pick(adamw32_kernel<RFX_F16, true, false>, adamw32_kernel<RFX_F16, true, true>); break;
        case 6: pick(adamw8_kernel<RFX_F32, false, false>, adamw8_kernel<RFX_F32, false, true>); break;
        case 7: pick(adamw8_kernel<RFX_BF16, false, false>, adamw8_kernel<RFX_BF16, false, true>); break;
        case 8: pick(adamw8_kernel<RFX_F16, false, false>, adamw8_kernel<RFX_F16, false, true>); break;
        case 10: pick(adamw8_kernel<RFX_BF16, true, false>, adamw8_kernel<RFX_BF16, true, true>); break;
        case 11: pick(adamw8_kernel<RFX_F16, true, false>, adamw8_kernel<RFX_F16, true, true>); break;
        default: return RFX_ERR_ARG;
    }
    void* args[] = {&k};
    RFX_HIP_TRY(hipLaunchKernel(kernel, dim3((unsigned)k.first[k.count]), dim3(AW_THREADS), args, 0, stream));
    RFX_LAUNCH_CHECK();
    k.count = 0;
    k.clip.norm32 = nullptr;                                               // the first launch has written it
    return RFX_OK;
}

static int kind_of(const rfx_adamw_tensor& t, const rfx_adamw_group& g) { return t.dtype + (t.master ? 3 : 0) + (g.state_bits == 8 ? 6 : 0); }

static bool tensor_ok(const rfx_adamw_tensor& t, const rfx_adamw_group* groups, int n_groups) {
    if (t.n < 0 || t.n > MOST_ELEMENTS || t.group < 0 || t.group >= n_groups || t.dtype < RFX_F32 || t.dtype > RFX_F16) return false;
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

// memory that a launch writes: no two of its tensors may share any.  Tensors mostly lie one behind the other, outside of all before
struct Written {
    uintptr_t from[GN_TENSORS], to[GN_TENSORS], least = ~(uintptr_t)0, most = 0;
    int count = 0;
    void clear() { count = 0; least = ~(uintptr_t)0; most = 0; }
    bool shares(const void* p, int64_t bytes) const {
        const uintptr_t a = (uintptr_t)p, b = a + (uintptr_t)bytes;
        if (a >= most || b <= least) return false;
        for (int i = 0; i < count; ++i)
            if (a < to[i] && from[i] < b) return true;
        return false;
    }
    void add(const void* p, int64_t bytes) {
        from[count] = (uintptr_t)p;
        to[count] = from[count] + (uintptr_t)bytes;
        least = from[count] < least ? from[count] : least;
        most = to[count] > most ? to[count] : most;
        ++count;
    }
};
static_assert(AW_TENSORS <= GN_TENSORS, "");

// gradients [at, at + as many as fit) as one launch, in at most `most` pieces where pieces of whole rounds allow it; returns how many
// were taken, 0: none left.  apart: no two of a launch share memory (they are written)
static int gather(const rfx_grad_tensor* t, int count, int& at, GnArgs& k, int most, bool apart) {
    Written written;
    int64_t all = 0;
    k.count = 0;
    for (; at < count && k.count < GN_TENSORS; ++at) {
        if (t[at].n == 0) continue;
        const int64_t size = t[at].n * elem_bytes(t[at].dtype);
        if (apart && written.shares(t[at].grad, size)) break;
        if (apart) written.add(t[at].grad, size);
        k.t[k.count].g = t[at].grad;
        k.t[k.count].n = t[at].n;
        k.dtype[k.count++] = (uint8_t)t[at].dtype;
        all += t[at].n;
    }
    const auto whole = [](int64_t n) { const int64_t r = n > 4 * GN_ROUND ? 4 * GN_ROUND : GN_ROUND; return (n + r - 1) / r * r; };
    const auto pieces_at = [&](int64_t piece) {                            // a remainder under an eighth is not worth a longer piece for all
        int64_t n = 0;
        for (int i = 0; i < k.count; ++i) n += (k.t[i].n + piece - 1 - piece / 8) / piece;
        return n;
    };
    int64_t piece = whole(all / most + 1);
    while (pieces_at(piece) > most && piece < (int64_t)1 << 30) piece = whole(piece + piece / 64 + 1);
    k.piece = (int)(piece < (int64_t)1 << 30 ? piece : (int64_t)1 << 30);
    int64_t pieces = 0;
    for (int i = 0; i < k.count; ++i) {
        k.first[i] = (int32_t)pieces;
        pieces += (k.t[i].n + k.piece - 1) / k.piece;
    }
    k.first[k.count] = k.pieces = (int32_t)pieces;
    return k.count;
}

static bool grads_ok(const rfx_grad_tensor* t, int count) {
    if (count < 0 || (count > 0 && !t)) return false;
    for (int i = 0; i < count; ++i) {
        if (t[i].n < 0 || t[i].n > MOST_ELEMENTS || t[i].dtype < RFX_F32 || t[i].dtype > RFX_F16) return false;
        if (t[i].n > 0 && (!t[i].grad || ((uintptr_t)t[i].grad & (uintptr_t)(elem_bytes(t[i].dtype) - 1)))) return false;
    }
    return true;
}

// Blocks of a step from which the partial results are joined in a launch of their own.  A clipped step, us (every wave / a launch), 32 bits:
// 0.1 million parameters 11.3 / 13.5, 2 million 17.4 / 17.6, 8 million 46.6 / 45.7, 40 million 194.7 / 192.8; 8 bits: 11.2 / 11.8,
// 16.6 / 16.7, 38.0 / 34.6, 158 / 139.
constexpr int64_t JOIN_BLOCKS = 2048;

static size_t partials(int count) { return (size_t)JOIN * ((count + GN_TENSORS - 1) / GN_TENSORS) + 2; }

// partial results of the norm; `from`: how a kernel finds the factor in them
static int norm_launches(const rfx_grad_tensor* tensors, int count, int max, double max_norm, double* workspace, int& n, ClipSource& from,
                         hipStream_t stream) {
    GnArgs k;
    n = 0;
    for (int at = 0; gather(tensors, count, at, k, JOIN, false) > 0;) {
        const int blocks = k.pieces < JOIN ? k.pieces : JOIN;
        k.partial = workspace + n;
        n += blocks;
        if (max) hipLaunchKernelGGL(grad_norm_kernel<true>, dim3(blocks), dim3(GN_THREADS), 0, stream, k);
        else hipLaunchKernelGGL(grad_norm_kernel<false>, dim3(blocks), dim3(GN_THREADS), 0, stream, k);
        RFX_LAUNCH_CHECK();
    }
    from = ClipSource{workspace, nullptr, max_norm, nullptr, n, max};
    return RFX_OK;
}

// ... joined beforehand where there are more than a block joins by itself, or many blocks that would
static int join(double* workspace, int n, int64_t blocks, float* norm32, ClipSource& from, hipStream_t stream) {
    from.norm32 = norm32;
    if (n <= JOIN && blocks <= JOIN_BLOCKS) return RFX_OK;
    hipLaunchKernelGGL(grad_norm_join_kernel, dim3(1), dim3(JOIN), 0, stream, workspace, n, from.max, from.max_norm, workspace + n, norm32);
    RFX_LAUNCH_CHECK();
    from = ClipSource{workspace, workspace + n, 0.0, nullptr, 0, 0};
    return RFX_OK;
}

// the norm of no element at all, which no other launch of the call has written
static int no_norm(const double* workspace, float* norm32, hipStream_t stream) {
    if (!norm32) return RFX_OK;
    hipLaunchKernelGGL(grad_norm_join_kernel, dim3(1), dim3(JOIN), 0, stream, workspace, 0, 0, 0.0, nullptr, norm32);
    RFX_LAUNCH_CHECK();
    return RFX_OK;
}

static int scale_launches(const rfx_grad_tensor* tensors, int count, ClipSource from, hipStream_t stream) {
    GnArgs k;
    for (int at = 0; gather(tensors, count, at, k, JOIN, true) > 0;) {
        k.clip = from;
        hipLaunchKernelGGL(grad_scale_kernel, dim3(k.pieces < JOIN ? k.pieces : JOIN), dim3(GN_THREADS), 0, stream, k);
        RFX_LAUNCH_CHECK();
        from.norm32 = nullptr;
    }
    return no_norm(from.partial, from.norm32, stream);
}

}  // namespace rfx

using namespace rfx;

extern "C" {

size_t rfx_adamw_tensor_bytes(void) { return sizeof(rfx_adamw_tensor); }
size_t rfx_adamw_group_bytes(void) { return sizeof(rfx_adamw_group); }
size_t rfx_adamw_workspace_bytes(int count) {
    return count > 0 ? ((size_t)count * sizeof(AwStep) + partials(count) * sizeof(double) + 15) / 16 * 16 : 0;
}

int rfx_adamw_step(const rfx_adamw_tensor* tensors, int count, const rfx_adamw_group* groups, int n_groups, const rfx_grad_tensor* clip_grads,
                   double max_norm, float* norm32, void* workspace, size_t workspace_bytes, rfx_stream stream) {
    if (count == 0) return RFX_OK;
    if (!tensors || count < 0 || !groups || n_groups < 1) return RFX_ERR_ARG;
    bool on_device = false;
    unsigned kinds = 0;
    int64_t bytes = 0, blocks_in_all = 0;
    for (int i = 0; i < n_groups; ++i)
        if (!group_ok(groups[i])) return RFX_ERR_ARG;
    for (int i = 0; i < count; ++i) {
        if (!tensor_ok(tensors[i], groups, n_groups)) return RFX_ERR_ARG;
        if (pieces_of(tensors[i].n) > AW_BLOCKS) return RFX_ERR_UNSUPPORTED;
        on_device |= tensors[i].step_dev != nullptr;
        kinds |= 1U << kind_of(tensors[i], groups[tensors[i].group]);
        bytes += tensors[i].n * (2 * elem_bytes(tensors[i].dtype) + (tensors[i].master ? 4 : 0) + (groups[tensors[i].group].state_bits == 8 ? 2 : 8));
        blocks_in_all += pieces_of(tensors[i].n);
    }
    if (clip_grads && (!grads_ok(clip_grads, count) || !(max_norm >= 0.0))) return RFX_ERR_ARG;
    if ((on_device || clip_grads) && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < rfx_adamw_workspace_bytes(count)))
        return RFX_ERR_WORKSPACE;
    const bool past = bytes >= STREAM_BYTES;
    AwArgs k;
    PrepArgs prep;
    prep.out = (AwStep*)workspace;
    k.clip = ClipSource{};
    if (clip_grads) {
        int n = 0;
        double* at = (double*)((char*)workspace + (size_t)count * sizeof(AwStep));
        int rc = norm_launches(clip_grads, count, 0, max_norm, at, n, k.clip, as_stream(stream));
        if (rc == RFX_OK) rc = join(at, n, blocks_in_all, norm32, k.clip, as_stream(stream));
        if (rc != RFX_OK) return rc;
    }
    for (int kind = 0; kind < 12; ++kind) {
        if (!(kinds >> kind & 1)) continue;
        for (int counted = 0; counted < 2; ++counted) {                    // step counts from the host, then those on the device
            if (counted && !on_device) break;
            int group_at[AW_GROUPS], used = 0;
            int64_t blocks = 0;
            Written written;
            k.count = 0;
            k.dev = nullptr;
            for (int i = 0; i <= count; ++i) {
                if (i < count) {
                    const rfx_adamw_tensor& t = tensors[i];
                    if (kind_of(t, groups[t.group]) != kind || (t.step_dev != nullptr) != (counted != 0)) continue;
                    if (t.n == 0 && !counted) continue;
                    const int64_t pieces = pieces_of(t.n);
                    int gi = 0;
                    while (gi < used && group_at[gi] != t.group) ++gi;
                    const int64_t size = t.n * elem_bytes(t.dtype);
                    if (k.count < AW_TENSORS && gi < AW_GROUPS && blocks + pieces <= AW_BLOCKS && !written.shares(t.param, size)) {
                        if (gi == used) {
                            const rfx_adamw_group& g = groups[t.group];
                            AwGroup& a = k.group[gi];
                            a.b1 = g.beta1; a.c1 = 1.0 - g.beta1; a.b2 = g.beta2; a.c2 = 1.0 - g.beta2;
                            a.eps = (float)g.eps;
                            if (g.state_bits == 8 && g.eps > 0.0) a.eps = fmaxf(a.eps, 0x1p-126f);      // rcp takes less for 0
                            a.wide = wide_from(a.eps);
                            a.sign = g.maximize ? -1.f : 1.f;
                            if (!counted) a.s = step_scalars(g.lr, g.beta1, g.beta2, g.weight_decay, (double)g.step, g.seed);
                            prep.g[gi] = {g.lr, g.beta1, g.beta2, g.weight_decay, g.lr_dev, g.seed};
                            group_at[used++] = t.group;
                        }
                        written.add(t.param, size);
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
                const int rc = adamw_launch(k, counted ? &prep : nullptr, kind, past, as_stream(stream));
                if (rc != RFX_OK) return rc;
                used = 0;
                blocks = 0;
                written.clear();
            }
        }
    }
    return no_norm(k.clip.partial, k.clip.norm32, as_stream(stream));
}

int rfx_adamw_moments(const rfx_moment_tensor* tensors, int count, rfx_stream stream) {
    if (count == 0) return RFX_OK;
    if (!tensors || count < 0) return RFX_ERR_ARG;
    int64_t bytes = 0;
    for (int i = 0; i < count; ++i) {
        const rfx_moment_tensor& t = tensors[i];
        if (t.n < 0 || t.n > MOST_ELEMENTS || (t.n > 0 && (!t.exp_avg || !t.exp_avg_sq || !t.exponents || !t.out_avg || !t.out_avg_sq))) return RFX_ERR_ARG;
        if (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq | (uintptr_t)t.out_avg | (uintptr_t)t.out_avg_sq) & 3) return RFX_ERR_ARG;
        if (pieces_of(t.n) > AW_BLOCKS) return RFX_ERR_UNSUPPORTED;
        bytes += 8 * t.n;                                                  // of the outputs: 332 MB of them 72 us plain, 61 past the caches
    }
    MomArgs k;
    for (int i = 0; i < count;) {
        int64_t blocks = 0;
        for (k.count = 0; i < count && k.count < AW_TENSORS; ++i) {
            if (tensors[i].n == 0) continue;
            const int64_t pieces = pieces_of(tensors[i].n);
            if (blocks + pieces > AW_BLOCKS) break;
            k.t[k.count] = tensors[i];
            k.first[k.count++] = (int32_t)blocks;
            blocks += pieces;
        }
        if (k.count == 0) break;
        k.first[k.count] = (int32_t)blocks;
        const auto kernel = bytes >= STREAM_BYTES ? adamw_moments_kernel<true> : adamw_moments_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(AW_THREADS), 0, as_stream(stream), k);
        RFX_LAUNCH_CHECK();
    }
    return RFX_OK;
}

size_t rfx_grad_norm_workspace_bytes(int count) { return count >= 0 ? partials(count) * sizeof(double) : 0; }

static int norm_args(const rfx_grad_tensor* tensors, int count, int norm_type, double max_norm, const void* workspace, size_t workspace_bytes) {
    if (!grads_ok(tensors, count) || !(max_norm >= 0.0)) return RFX_ERR_ARG;
    if (norm_type != 2 && norm_type != 0) return RFX_ERR_UNSUPPORTED;
    return !workspace || ((uintptr_t)workspace & 7) || workspace_bytes < rfx_grad_norm_workspace_bytes(count) ? RFX_ERR_WORKSPACE : RFX_OK;
}

int rfx_grad_norm(const rfx_grad_tensor* tensors, int count, int norm_type, double max_norm, double* clip, float* norm32,
                  void* workspace, size_t workspace_bytes, rfx_stream stream) {
    if (!clip || ((uintptr_t)clip & 7)) return RFX_ERR_ARG;
    int rc = norm_args(tensors, count, norm_type, max_norm, workspace, workspace_bytes), n = 0;
    if (rc != RFX_OK) return rc;
    ClipSource from;
    rc = norm_launches(tensors, count, norm_type == 0, max_norm, (double*)workspace, n, from, as_stream(stream));
    if (rc != RFX_OK) return rc;
    hipLaunchKernelGGL(grad_norm_join_kernel, dim3(1), dim3(JOIN), 0, as_stream(stream), (const double*)workspace, n, from.max, max_norm, clip,
                       norm32);
    RFX_LAUNCH_CHECK();
    return RFX_OK;
}

int rfx_grad_scale(const rfx_grad_tensor* tensors, int count, const double* clip, rfx_stream stream) {
    if (!grads_ok(tensors, count) || !clip || ((uintptr_t)clip & 7)) return RFX_ERR_ARG;
    return scale_launches(tensors, count, ClipSource{nullptr, clip, 0.0, nullptr, 0, 0}, as_stream(stream));
}

int rfx_grad_clip(const rfx_grad_tensor* tensors, int count, int norm_type, double max_norm, float* norm32, void* workspace,
                  size_t workspace_bytes, rfx_stream stream) {
    int rc = norm_args(tensors, count, norm_type, max_norm, workspace, workspace_bytes), n = 0;
    if (rc != RFX_OK) return rc;
    ClipSource from;
    rc = norm_launches(tensors, count, norm_type == 0, max_norm, (double*)workspace, n, from, as_stream(stream));
    if (rc == RFX_OK) rc = join((double*)workspace, n, 0, norm32, from, as_stream(stream));
    if (rc != RFX_OK) return rc;
    return scale_launches(tensors, count, from, as_stream(stream));
}

}  // extern "C"
