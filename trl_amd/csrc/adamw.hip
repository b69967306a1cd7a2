// K9: one AdamW step over many tensors, with the global gradient norm clipped, both moments in fp32 or in 8 bits.
//
//   c = min(1, max_norm / (|g| + 1e-6)), |g| over all tensors;  m' = b1 m + (1 - b1) c g;  v' = b2 v + (1 - b2) (c g)^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Elementwise and HBM bound: parameter and moments are read and written once, the gradient read once, and once more for the norm,
// which has to be known first.  Three kinds of launches: partial sums of squares (64 bits), one workgroup that adds them and
// moves every tensor's step counter on (so that a captured step counts when it is replayed), the update.  Tensors come as tables
// in the kernels' arguments: nothing is copied to the device, and a captured graph holds its own.  Measured on 355M entries: norm 229 us in
// fp32 (6.2 TB/s), 118 in bf16 (6.0); update 1560 to 1720 us in fp32 with fp32 moments (5.8 to 6.4 TB/s, from box to box), 395 to 405 for 117M in
// bf16 (6.3 to 6.5), 660 to 770 in bf16
// with 8-bit moments (4.6 to 5.4: the hash and the rounding take as long as the memory).  With adapters, 224 tensors of 8192 to 81920
// entries in fp32, the five launches' beginnings and ends are a third of the 66 us.
//
// 8-bit moments: blocks of 256 entries with a power-of-two scale that takes the block's largest entry to at most 448.  m has a
// sign, 4 bits of exponent and 3 of mantissa (the OCP e4m3 format); v, which is not negative, 4 and 4 and keeps a code over 0
// where it is not 0, because its root is divided by.  A step moves v by 1 - b2 of itself, 0.1 % with the usual 0.999, and codes
// are 3 to 6 % apart: rounding to the nearest would leave v where it is for good.  So the rounding is stochastic, up with the
// probability that keeps the mean; its 16 random bits per moment are a hash of seed, step, tensor and entry, and the same call
// gives the same bits.  The arithmetic of the moments is that of separate fp32 products and sums, in a fixed order.
#include <math.h>

#include "common.hpp"

namespace trlk {
namespace {

constexpr int kThreads = 256;
constexpr int kStateBlock = 256;         // entries that share a scale
constexpr int kNormChunk = 8192;         // entries of a workgroup of the norm
constexpr int kChunk = 2048;             // entries of a workgroup of the update: adapters of 40000 entries fill the chip, too
constexpr int kTable32 = 83;             // tensors of an update launch with fp32 moments  (4 KB of arguments)
constexpr int kTable8 = 62;              // with 8-bit moments                             (4 KB)
constexpr int kNormTable = 250;          // pieces of tensors of a norm launch             (4 KB)
constexpr int64_t kNormPiece = int64_t(1) << 31;
constexpr int64_t kMaxGroups = (int64_t(1) << 32) / kThreads - 1;  // of a launch: it has fewer than 2^32 threads
constexpr int64_t kMaxNumel = int64_t(1) << 34;
static_assert(kMaxNumel / kChunk <= kMaxGroups && kNormPiece / kNormChunk <= kMaxGroups, "a tensor, or a piece of one, fits into a launch");
constexpr int kStepTable = 240;          // tensors of a launch of the step counters

// ---- scalars that the update reads: one record per tensor -------------------------------------------------------------
struct alignas(16) Scalars {
    float beta1, one_minus_beta1, beta2, one_minus_beta2;
    float size, inv_sqrt_bc2, eps, decay;
    uint32_t salt, pad[3];
};
struct alignas(16) Header {
    float clip, norm, pad[2];
};

// Loads and stores of what a step touches once, past the caches: a step of 355M fp32 entries with fp32 moments 1.98 ms instead of 2.14, of 117M in
// bf16 481 us instead of 544, both sides in turn (the norm's loads are plain: the update reads the gradients again).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename V>
__device__ __forceinline__ V once(const void* p) {
    return __builtin_nontemporal_load(static_cast<const V*>(p));
}
template <typename V>
__device__ __forceinline__ void once(void* p, V v) {
    __builtin_nontemporal_store(v, static_cast<V*>(p));
}

// A 32-bit hash: xor with the upper half, multiply, twice (the multipliers: best of 400 random odd pairs in how evenly one
// flipped bit flips the others).
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x55CE65ADu;
    x = (x ^ (x >> 15)) * 0xCDBE2AF7u;
    return x ^ (x >> 16);
}

// ---- norm ------------------------------------------------------------------------------------------------------------
struct NormEntry {
    const void* grad;
    uint32_t numel;
    uint32_t first : 31, aligned : 1;  // first workgroup of the launch; whether the data is 16-byte aligned
};
struct NormTable {
    NormEntry e[kNormTable];
    int32_t n;
    double* partial;  // one per workgroup
};

// the entry of workgroup w in a table that is sorted by `first`
template <typename E>
__device__ __forceinline__ int entry_of(const E* e, int n, uint32_t w) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (e[mid].first <= w) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void norm_kernel(NormTable t) {
    typedef typename Elem<DT>::type T;
    constexpr int EPV = Elem<DT>::EPV;
    __shared__ double scratch[kThreads / kWave];
    const int i = entry_of(t.e, t.n, blockIdx.x);
    const int64_t begin = int64_t(blockIdx.x - t.e[i].first) * kNormChunk, end = begin + kNormChunk < t.e[i].numel ? begin + kNormChunk : t.e[i].numel;
    const T* g = static_cast<const T*>(t.e[i].grad);
    double s = 0.0;
    int64_t e = begin;
    if (t.e[i].aligned) {
        const int64_t whole = begin + (end - begin) / EPV * EPV;
        constexpr int U = 4;  // loads in flight
        for (int64_t at = begin + threadIdx.x * EPV; at < whole; at += U * kThreads * EPV) {
            u32x4 q[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int64_t to = at + j * kThreads * EPV;
                q[j] = to < whole ? *reinterpret_cast<const u32x4*>(g + to) : u32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                float x[EPV];
                Elem<DT>::unpack(q[j], x);
#pragma unroll
                for (int k = 0; k < EPV; ++k) s = __builtin_fma(double(x[k]), double(x[k]), s);
            }
        }
        e = whole;
    }
    for (int64_t at = e + threadIdx.x; at < end; at += kThreads) {
        const double x = double(Elem<DT>::load1(g + at));
        s = __builtin_fma(x, x, s);
    }
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double r = 0.0;
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) r += scratch[w];
        t.partial[blockIdx.x] = r;
    }
}

// ---- norm and step counters ------------------------------------------------------------------------------------------
struct StepEntry {
    float* step;
    uint32_t index, pad;
};
struct StepTable {
    StepEntry e[kStepTable];
    int32_t n;
    uint32_t seed;
    double lr, beta1, beta2, eps, weight_decay;
    double log2_beta1, log2_beta2;
    const float* d_lr;
    Scalars* scalars;
    const double* partial;  // null: this launch does not add up the norm
    int64_t n_partial;
    double max_norm;        // not over 0: no clipping
    Header* header;
    float* out_norm;
};

__global__ __launch_bounds__(1024) void step_kernel(StepTable t) {
    __shared__ double scratch[1024 / kWave];
    for (int i = threadIdx.x; i < t.n; i += 1024) {
        const float now = *t.e[i].step + 1.f;
        *t.e[i].step = now;
        const double lr = t.d_lr ? double(*t.d_lr) : t.lr;
        Scalars s{};
        s.beta1 = float(t.beta1);
        s.one_minus_beta1 = float(1.0 - t.beta1);
        s.beta2 = float(t.beta2);
        s.one_minus_beta2 = float(1.0 - t.beta2);
        s.size = float(lr / (1.0 - exp2(t.log2_beta1 * double(now))));
        s.inv_sqrt_bc2 = float(1.0 / sqrt(1.0 - exp2(t.log2_beta2 * double(now))));
        s.eps = float(t.eps);
        s.decay = float(1.0 - lr * t.weight_decay);
        s.salt = mix(mix(uint32_t(int64_t(now)) ^ t.seed) + 0x9E3779B9u * (t.e[i].index + 1u));
        t.scalars[t.e[i].index] = s;
    }
    if (!t.header) return;
    double sum = 0.0;
    constexpr int U = 8;  // loads in flight
    for (int64_t i = threadIdx.x; i < t.n_partial; i += U * 1024) {
        double x[U];
#pragma unroll
        for (int j = 0; j < U; ++j) x[j] = i + j * 1024 < t.n_partial ? t.partial[i + j * 1024] : 0.0;
#pragma unroll
        for (int j = 0; j < U; ++j) sum += x[j];
    }
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    double r = 0.0;
#pragma unroll
    for (int w = 0; w < 1024 / kWave; ++w) r += scratch[w];
    const double norm = sqrt(r), clip = t.max_norm / (norm + 1e-6);
    t.header->norm = float(norm);
    t.header->clip = t.max_norm > 0.0 && !(clip >= 1.0) ? float(clip) : 1.f;  // (a NaN goes on to the parameters)
    if (t.out_norm) *t.out_norm = float(norm);
}

// ---- update ----------------------------------------------------------------------------------------------------------
template <int BITS>
struct UpdateEntry {
    void* param;
    const void* grad;
    void *exp_avg, *exp_avg_sq;
    int64_t numel;
    uint32_t first;
    uint32_t index : 31, aligned : 1;
};
template <>
struct UpdateEntry<8> : UpdateEntry<32> {
    float *exp_avg_scale, *exp_avg_sq_scale;
};
template <int BITS>
struct UpdateTable {
    static constexpr int kSize = BITS == 32 ? kTable32 : kTable8;
    UpdateEntry<BITS> e[kSize];
    int32_t n;
    const Scalars* scalars;
    const Header* header;  // null: no clipping
};

// the moments after a step, in the order of operations that the header names
__device__ __forceinline__ void moments(const Scalars& s, float clip, float g, float& m, float& v) {
#pragma clang fp contract(off)
    g = g * clip;
    const float a = m * s.beta1, b = g * s.one_minus_beta1;
    m = a + b;
    const float c = v * s.beta2, d = g * g, e = d * s.one_minus_beta2;
    v = c + e;
}
// The hardware's root and reciprocal, each good to a unit of the last place, save that the root of a subnormal number is 0 and the reciprocal of
// one infinite.  TINY scales both away from there, by powers of two; it is for an eps that does not hide the root of a subnormal number:
// that is under 2^-63, and with eps >= 2^-38 / sqrt(1 - b2^t) it changes the divisor by less than 2^-25 of itself.
template <bool TINY>
__device__ __forceinline__ float updated(const Scalars& s, float p, float m, float v) {
    if constexpr (TINY) {
        const bool low = v < 0x1p-96f;
        const float root = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v) * (low ? 0x1p-32f : 1.f);
        const float d = fmaf(root, s.inv_sqrt_bc2, s.eps), up = d < 0x1p-64f ? 0x1p64f : 1.f;
        return fmaf(-s.size, (m * up) * __builtin_amdgcn_rcpf(d * up), p * s.decay);
    }
    const float d = fmaf(__builtin_amdgcn_sqrtf(v), s.inv_sqrt_bc2, s.eps);
    return fmaf(-s.size, m * __builtin_amdgcn_rcpf(d), p * s.decay);
}
template <int N>
__device__ __forceinline__ void update_n(const Scalars& s, const float (&m)[N], const float (&v)[N], float (&x)[N]) {
    if (s.eps < s.inv_sqrt_bc2 * 0x1p-38f) {  // (the same for a whole tensor)
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = updated<true>(s, x[k], m[k], v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = updated<false>(s, x[k], m[k], v[k]);
    }
}

// N entries at `at`, all of them or those before `n`
template <int DT, int N>
__device__ __forceinline__ void load_n(const typename Elem<DT>::type* p, int64_t at, int64_t n, bool whole, float (&x)[N]) {
    constexpr int EPV = Elem<DT>::EPV;
    if (whole) {
        if constexpr (N >= EPV) {
#pragma unroll
            for (int i = 0; i < N / EPV; ++i) Elem<DT>::unpack(once<u32x4>(p + at + i * EPV), x + i * EPV);
        } else {  // 4 entries of a 16-bit type
            const u32x2 q = once<u32x2>(p + at);
            Elem<DT>::unpack2(q.x, x);
            Elem<DT>::unpack2(q.y, x + 2);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = at + k < n ? Elem<DT>::load1(p + at + k) : 0.f;
    }
}
template <int DT, int N>
__device__ __forceinline__ void store_n(typename Elem<DT>::type* p, int64_t at, int64_t n, bool whole, const float (&x)[N]) {
    constexpr int EPV = Elem<DT>::EPV;
    if (whole) {
        if constexpr (N >= EPV) {
#pragma unroll
            for (int i = 0; i < N / EPV; ++i) once(p + at + i * EPV, Elem<DT>::pack(x + i * EPV));
        } else {
            once(p + at, u32x2{Elem<DT>::pack2(x[0], x[1]), Elem<DT>::pack2(x[2], x[3])});
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (at + k < n) Elem<DT>::store1(p + at + k, x[k]);
    }
}

// ---- 8-bit floats -----------------------------------------------------------------------------------------------------
// The bits of a code, moved to where an fp32 has them, are the value times 2^-120 (the biases are 7 and 127; codes of exponent 0
// become subnormal numbers, which count here).
template <int MANT>
__device__ __forceinline__ float decode8(uint32_t c) {
    if constexpr (MANT == 3)
        return __uint_as_float((c & 0x7fu) << 20 | (c & 0x80u) << 24) * 0x1p120f;
    else
        return __uint_as_float(c << 19) * 0x1p120f;
}
// the four e4m3 codes of a word: the hardware knows the format
__device__ __forceinline__ void decode_e4m3(uint32_t w, float* x) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
// the lowest bytes of four words
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t* c) {
    const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// code of y >= 0, 448 at most, rounded up where the dropped part and 16 random bits exceed one step
template <int MANT>
__device__ __forceinline__ uint32_t encode8(float y, uint32_t r16) {
    constexpr int shift = 23 - MANT;
    const uint32_t normal = ((__float_as_uint(y) + (r16 << (shift - 16))) >> shift) - (120u << MANT);
    const uint32_t small = (uint32_t(y * float(1 << (22 + MANT))) + r16) >> 16;
    return y < 0x1p-6f ? small : normal;
}
// power-of-two scale that takes `largest` to (224, 448], and its inverse; 1 for a block of zeros, NaN where it is not finite
__device__ __forceinline__ void block_scale(float largest, float& scale, float& inverse) {
    const uint32_t word = __float_as_uint(largest);
    int power = int(word >> 23) - 135 + ((word & 0x7fffffu) > 0x600000u ? 1 : 0);
    power = power < -126 ? -126 : power;
    scale = __uint_as_float(uint32_t(power + 127) << 23);
    inverse = __uint_as_float(uint32_t(127 - power) << 23);
    if (largest == 0.f) scale = inverse = 1.f;
    if (!(largest < INFINITY)) {
        scale = NAN;
        inverse = 0.f;
    }
}
__device__ __forceinline__ float half_wave_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = __builtin_elementwise_maximum(v, __shfl_xor(v, o));
    return v;
}

template <int DT, int BITS>
__global__ __launch_bounds__(kThreads) void update_kernel(UpdateTable<BITS> t) {
    typedef typename Elem<DT>::type T;
    const int i = entry_of(t.e, t.n, blockIdx.x);
    const UpdateEntry<BITS>& en = t.e[i];
    const Scalars s = t.scalars[en.index];
    const float clip = t.header ? t.header->clip : 1.f;
    const int64_t n = en.numel, begin = int64_t(blockIdx.x - en.first) * kChunk;
    T* p = static_cast<T*>(en.param);
    const T* g = static_cast<const T*>(en.grad);
    constexpr int N = BITS == 32 ? 4 : 8;
    for (int64_t at = begin + threadIdx.x * N; at < begin + kChunk; at += kThreads * N) {
        if constexpr (BITS == 32) {
            if (at >= n) break;
        } else {
            if (at / kStateBlock * kStateBlock >= n) break;  // (a half wave is in a block together)
        }
        const bool whole = en.aligned && at + N <= n;
        float x[N], y[N], m[N], v[N];
        load_n<DT, N>(p, at, n, whole, x);
        load_n<DT, N>(g, at, n, whole, y);
        if constexpr (BITS == 32) {
            float *pm = static_cast<float*>(en.exp_avg), *pv = static_cast<float*>(en.exp_avg_sq);
            load_n<TRLK_F32, N>(pm, at, n, whole, m);
            load_n<TRLK_F32, N>(pv, at, n, whole, v);
#pragma unroll
            for (int k = 0; k < N; ++k) moments(s, clip, y[k], m[k], v[k]);
            update_n(s, m, v, x);
            store_n<DT, N>(p, at, n, whole, x);
            store_n<TRLK_F32, N>(pm, at, n, whole, m);
            store_n<TRLK_F32, N>(pv, at, n, whole, v);
        } else {
            uint8_t *pm = static_cast<uint8_t*>(en.exp_avg), *pv = static_cast<uint8_t*>(en.exp_avg_sq);
            const int64_t block = at / kStateBlock;
            const float sm = en.exp_avg_scale[block], sv = en.exp_avg_sq_scale[block];
            uint32_t cm[2] = {0, 0}, cv[2] = {0, 0};
            if (whole) {
                const u32x2 a = once<u32x2>(pm + at), b = once<u32x2>(pv + at);
                cm[0] = a.x, cm[1] = a.y, cv[0] = b.x, cv[1] = b.y;
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    if (at + k < n) {
                        cm[k / 4] |= uint32_t(pm[at + k]) << (8 * (k % 4));
                        cv[k / 4] |= uint32_t(pv[at + k]) << (8 * (k % 4));
                    }
                }
            }
            decode_e4m3(cm[0], m);
            decode_e4m3(cm[1], m + 4);
            float am = 0.f, av = 0.f;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                m[k] *= sm;
                v[k] = decode8<4>(cv[k / 4] >> (8 * (k % 4)) & 0xffu) * sv;
                moments(s, clip, y[k], m[k], v[k]);
                if (whole || at + k < n) {
                    am = __builtin_elementwise_maximum(am, fabsf(m[k]));
                    av = __builtin_elementwise_maximum(av, v[k]);
                }
            }
            update_n(s, m, v, x);
            store_n<DT, N>(p, at, n, whole, x);
            am = half_wave_max(am);
            av = half_wave_max(av);
            float nm, nv, im, iv;
            block_scale(am, nm, im);
            block_scale(av, nv, iv);
            uint32_t em[N], ev[N];  // (of a block that is not finite any bytes: its scale is NaN)
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const uint32_t r = mix(s.salt + uint32_t(at + k) * 0x9E3779B1u);
                const float yv = v[k] * iv;
                em[k] = encode8<3>(fabsf(m[k]) * im, r & 0xffffu) | (m[k] < 0.f ? 0x80u : 0u);
                ev[k] = encode8<4>(yv, r >> 16);
                ev[k] = yv > 0.f && ev[k] == 0 ? 1u : ev[k];
            }
            cm[0] = pack_bytes(em), cm[1] = pack_bytes(em + 4), cv[0] = pack_bytes(ev), cv[1] = pack_bytes(ev + 4);
            if (whole) {
                once(pm + at, u32x2{cm[0], cm[1]});
                once(pv + at, u32x2{cv[0], cv[1]});
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    if (at + k < n) {
                        pm[at + k] = uint8_t(cm[k / 4] >> (8 * (k % 4)));
                        pv[at + k] = uint8_t(cv[k / 4] >> (8 * (k % 4)));
                    }
                }
            }
            if ((threadIdx.x & 31) == 0) {
                en.exp_avg_scale[block] = nm;
                en.exp_avg_sq_scale[block] = nv;
            }
        }
    }
}

// ---- the values of codes ---------------------------------------------------------------------------------------------
template <int MANT>
__global__ __launch_bounds__(kThreads) void state_values_kernel(const uint8_t* codes, const float* scales, int64_t n, uint16_t* out, int aligned) {
    const int64_t at = (int64_t(blockIdx.x) * kThreads + threadIdx.x) * 8;
    if (at >= n) return;
    const float s = scales[at / kStateBlock];
    if (aligned && at + 8 <= n) {
        const u32x2 c = once<u32x2>(codes + at);
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = decode8<MANT>((k < 4 ? c.x : c.y) >> (8 * (k % 4)) & 0xffu) * s;
        once(out + at, Elem<TRLK_BF16>::pack(x));
    } else {
        for (int k = 0; k < 8 && at + k < n; ++k) Elem<TRLK_BF16>::store1(out + at + k, decode8<MANT>(codes[at + k]) * s);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int64_t chunks(int64_t n, int64_t c) { return (n + c - 1) / c; }
size_t up16(size_t n) { return (n + 15) / 16 * 16; }

int64_t norm_groups(const trlk_adamw_tensor* t, int32_t n) {
    int64_t sum = 0;
    for (int32_t i = 0; i < n; ++i) sum += chunks(t[i].numel, kNormChunk);
    return sum;
}
void launch_norm(int dtype, const NormTable& t, unsigned grid, hipStream_t stream) {
    if (dtype == TRLK_F32) norm_kernel<TRLK_F32><<<grid, kThreads, 0, stream>>>(t);
    else if (dtype == TRLK_BF16) norm_kernel<TRLK_BF16><<<grid, kThreads, 0, stream>>>(t);
    else norm_kernel<TRLK_F16><<<grid, kThreads, 0, stream>>>(t);
}
// the update of the tensors of one type with moments of one kind
template <int DT, int BITS>
void update(const trlk_adamw_tensor* tensors, int32_t n_tensors, const Scalars* scalars, const Header* header, hipStream_t stream) {
    UpdateTable<BITS> t;
    t.n = 0;
    t.scalars = scalars;
    t.header = header;
    int64_t grid = 0;
    const auto flush = [&] {
        if (t.n) update_kernel<DT, BITS><<<unsigned(grid), kThreads, 0, stream>>>(t);
        t.n = 0;
        grid = 0;
    };
    for (int32_t i = 0; i < n_tensors; ++i) {
        const trlk_adamw_tensor& x = tensors[i];
        if (x.dtype != DT || x.state_bits != BITS || x.numel == 0) continue;
        const int64_t need = chunks(x.numel, kChunk);
        if (t.n == UpdateTable<BITS>::kSize || grid + need > kMaxGroups) flush();
        const size_t state_align = BITS == 32 ? 16 : 8, value_align = BITS == 32 && DT != TRLK_F32 ? 8 : 16;
        UpdateEntry<BITS>& e = t.e[t.n++];
        e.param = x.d_param, e.grad = x.d_grad, e.exp_avg = x.d_exp_avg, e.exp_avg_sq = x.d_exp_avg_sq;
        if constexpr (BITS == 8) e.exp_avg_scale = x.d_exp_avg_scale, e.exp_avg_sq_scale = x.d_exp_avg_sq_scale;
        e.numel = x.numel, e.first = uint32_t(grid), e.index = uint32_t(i);
        e.aligned = aligned_to(x.d_param, value_align) && aligned_to(x.d_grad, value_align) && aligned_to(x.d_exp_avg, state_align) &&
                    aligned_to(x.d_exp_avg_sq, state_align);
        grid += need;
    }
    flush();
}

int check_adamw(const trlk_adamw_tensor* t, int32_t n, const trlk_adamw_group* g, int32_t n_groups) {
    TRLK_REQUIRE(n >= 0 && n_groups >= 0 && (n == 0 || (t && g)), TRLK_ERR_NULL_POINTER, "adamw: null table");
    for (int32_t i = 0; i < n_groups; ++i) {
        TRLK_REQUIRE(g[i].beta1 >= 0.0 && g[i].beta1 < 1.0 && g[i].beta2 >= 0.0 && g[i].beta2 < 1.0, TRLK_ERR_BAD_VALUE,
                     "adamw: betas must be in [0, 1)");
        TRLK_REQUIRE(g[i].eps >= 0.0 && g[i].weight_decay >= 0.0 && (g[i].d_lr || g[i].lr >= 0.0), TRLK_ERR_BAD_VALUE,
                     "adamw: lr, eps and weight_decay must not be negative");
    }
    for (int32_t i = 0; i < n; ++i) {
        TRLK_REQUIRE(t[i].numel >= 0 && t[i].numel <= kMaxNumel, TRLK_ERR_BAD_SHAPE, "adamw: tensor %d has %lld entries", i, (long long)t[i].numel);
        TRLK_REQUIRE(t[i].dtype == TRLK_F32 || t[i].dtype == TRLK_BF16 || t[i].dtype == TRLK_F16, TRLK_ERR_BAD_DTYPE, "adamw: tensor %d: unsupported dtype %d", i, t[i].dtype);
        TRLK_REQUIRE(t[i].state_bits == 32 || t[i].state_bits == 8, TRLK_ERR_BAD_VALUE, "adamw: tensor %d: state_bits must be 8 or 32", i);
        TRLK_REQUIRE(t[i].group >= 0 && t[i].group < n_groups, TRLK_ERR_BAD_VALUE, "adamw: tensor %d is in no group", i);
        TRLK_REQUIRE(t[i].d_step && (t[i].numel == 0 || (t[i].d_param && t[i].d_grad && t[i].d_exp_avg && t[i].d_exp_avg_sq)), TRLK_ERR_NULL_POINTER,
                     "adamw: tensor %d: null operand", i);
        TRLK_REQUIRE(t[i].state_bits == 32 || t[i].numel == 0 || (t[i].d_exp_avg_scale && t[i].d_exp_avg_sq_scale), TRLK_ERR_NULL_POINTER, "adamw: tensor %d: null scales", i);
        const size_t es = elem_size(t[i].dtype), ss = t[i].state_bits == 32 ? 4 : 1;
        TRLK_REQUIRE(aligned_to(t[i].d_param, es) && aligned_to(t[i].d_grad, es) && aligned_to(t[i].d_exp_avg, ss) && aligned_to(t[i].d_exp_avg_sq, ss),
                     TRLK_ERR_BAD_STRIDE, "adamw: tensor %d: misaligned operand", i);
    }
    return TRLK_OK;
}

}  // namespace
}  // namespace trlk

using namespace trlk;

extern "C" size_t trlk_adamw_workspace_bytes(const trlk_adamw_tensor* tensors, int32_t n_tensors) {
    if (!tensors || n_tensors <= 0) return sizeof(Header);
    return sizeof(Header) + sizeof(Scalars) * size_t(n_tensors) + up16(sizeof(double) * size_t(norm_groups(tensors, n_tensors)));
}

extern "C" int trlk_adamw_step(const trlk_adamw_tensor* tensors, int32_t n_tensors, const trlk_adamw_group* groups, int32_t n_groups,
                               double max_grad_norm, uint32_t seed, float* d_out_norm, void* d_workspace, size_t workspace_bytes,
                               trlk_stream_t stream_) {
    clear_error();
    if (const int rc = check_adamw(tensors, n_tensors, groups, n_groups)) return rc;
    TRLK_REQUIRE(max_grad_norm == max_grad_norm, TRLK_ERR_BAD_VALUE, "adamw: max_grad_norm is NaN");
    const bool with_norm = max_grad_norm > 0.0 || d_out_norm != nullptr;
    if (n_tensors == 0 && !with_norm) return TRLK_OK;
    TRLK_REQUIRE(d_workspace && workspace_bytes >= trlk_adamw_workspace_bytes(tensors, n_tensors), TRLK_ERR_WORKSPACE, "adamw: workspace too small");
    TRLK_REQUIRE(aligned_to(d_workspace, 16), TRLK_ERR_WORKSPACE, "adamw: misaligned workspace");
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    Header* header = static_cast<Header*>(d_workspace);
    Scalars* scalars = reinterpret_cast<Scalars*>(header + 1);
    double* partial = reinterpret_cast<double*>(scalars + n_tensors);

    // sums of squares
    int64_t n_partial = 0;
    if (with_norm) {
        for (int dtype : {int(TRLK_F32), int(TRLK_BF16), int(TRLK_F16)}) {
            NormTable t;
            t.n = 0;
            t.partial = partial + n_partial;
            int64_t grid = 0;
            const auto flush = [&] {
                if (t.n) launch_norm(dtype, t, unsigned(grid), stream);
                n_partial += grid;
                t.n = 0;
                t.partial = partial + n_partial;
                grid = 0;
            };
            for (int32_t i = 0; i < n_tensors; ++i) {
                if (tensors[i].dtype != dtype) continue;
                for (int64_t at = 0; at < tensors[i].numel; at += kNormPiece) {
                    const int64_t n = tensors[i].numel - at < kNormPiece ? tensors[i].numel - at : kNormPiece, need = chunks(n, kNormChunk);
                    const char* g = static_cast<const char*>(tensors[i].d_grad) + at * int64_t(elem_size(dtype));
                    if (t.n == kNormTable || grid + need > kMaxGroups) flush();
                    NormEntry& e = t.e[t.n++];
                    e.grad = g, e.numel = uint32_t(n), e.first = uint32_t(grid), e.aligned = aligned_to(g, 16);
                    grid += need;
                }
            }
            flush();
        }
    }
    // step counters and scalars, a group at a time; the norm with the first of them
    bool norm_done = !with_norm;
    for (int32_t g = 0; g < n_groups || !norm_done; ++g) {
        StepTable t;
        t.n = 0;
        t.seed = seed;
        const trlk_adamw_group none{0.0, 0.0, 0.0, 0.0, 0.0, nullptr};
        const trlk_adamw_group& gr = g < n_groups ? groups[g] : none;
        t.lr = gr.lr, t.beta1 = gr.beta1, t.beta2 = gr.beta2, t.eps = gr.eps, t.weight_decay = gr.weight_decay, t.d_lr = gr.d_lr;
        t.log2_beta1 = log2(gr.beta1), t.log2_beta2 = log2(gr.beta2);  // (0: -inf, and its power 0)
        t.scalars = scalars;
        t.partial = partial;
        t.n_partial = n_partial;
        t.max_norm = max_grad_norm;
        t.out_norm = d_out_norm;
        const auto flush = [&] {
            t.header = norm_done ? nullptr : header;
            if (t.n || !norm_done) step_kernel<<<1, 1024, 0, stream>>>(t);
            norm_done = true;
            t.n = 0;
        };
        for (int32_t i = 0; i < n_tensors; ++i) {
            if (tensors[i].group != g) continue;
            if (t.n == kStepTable) flush();
            t.e[t.n++] = StepEntry{tensors[i].d_step, uint32_t(i), 0u};
        }
        flush();
    }
    const Header* clip = with_norm ? header : nullptr;
    update<TRLK_F32, 32>(tensors, n_tensors, scalars, clip, stream);
    update<TRLK_BF16, 32>(tensors, n_tensors, scalars, clip, stream);
    update<TRLK_F16, 32>(tensors, n_tensors, scalars, clip, stream);
    update<TRLK_F32, 8>(tensors, n_tensors, scalars, clip, stream);
    update<TRLK_BF16, 8>(tensors, n_tensors, scalars, clip, stream);
    update<TRLK_F16, 8>(tensors, n_tensors, scalars, clip, stream);
    return launch_status("adamw");
}

extern "C" int trlk_adamw_state_values(const uint8_t* d_codes, const float* d_scales, int64_t n, int32_t has_sign, void* d_out_bf16, trlk_stream_t stream) {
    clear_error();
    TRLK_REQUIRE(n >= 0 && n <= kMaxNumel, TRLK_ERR_BAD_SHAPE, "adamw_state_values: bad size %lld", (long long)n);
    if (n == 0) return TRLK_OK;
    TRLK_REQUIRE(d_codes && d_scales && d_out_bf16, TRLK_ERR_NULL_POINTER, "adamw_state_values: null operand");
    TRLK_REQUIRE(aligned_to(d_out_bf16, 2), TRLK_ERR_BAD_STRIDE, "adamw_state_values: misaligned output");
    const int al = aligned_to(d_codes, 8) && aligned_to(d_out_bf16, 16) ? 1 : 0;
    const dim3 grid(unsigned(chunks(n, kThreads * 8)));
    if (has_sign)
        state_values_kernel<3><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(d_codes, d_scales, n, static_cast<uint16_t*>(d_out_bf16), al);
    else
        state_values_kernel<4><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(d_codes, d_scales, n, static_cast<uint16_t*>(d_out_bf16), al);
    return launch_status("adamw_state_values");
}
