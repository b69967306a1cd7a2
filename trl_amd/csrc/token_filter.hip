// K8: tokens drawn from, and scored under, softmax(logits / T) after top-k, top-p and min-p.
//
// Order of a row's tokens: logit descending, index ascending.  All three filters keep a prefix of that order (top-k the first k,
// top-p those before which less than top_p of the mass lies that top-k kept, min-p those of weight >= min_p, the largest being 1),
// so what a row keeps is one border: a value, and among the tokens of exactly that value the last index.  With
// w_v = exp((x_v - max) / T) for the kept tokens, a token is drawn as the first index whose cumulative weight exceeds u * W.
//
// Two launches or four, and one for the gradient.  filter_scan_kernel reads the logits once, a wave per chunk of 2048, and leaves the chunk's
// maximum, its sum of weights in 64 bits and the maximum of every block of 64 logits.  filter_select_kernel has one workgroup per row:
// the block maxima bound the border from below (the k-th largest of them is at most the k-th largest logit; blocks whose maxima hold
// top_p of the mass hold the tokens of top-p), so that only blocks with a maximum over that bound are read again -- a few dozen of
// some thousand.  What comes after goes by the number of candidates in them: up to 128 are compared pair by pair; of up to 4096 the border
// is found in bins of distances from the maximum and then among the pairs of its bin, the token in its chunk; with more, without top-k,
// the row is passed over twice more (a count in bins; exact sums, chunk by chunk, before the border's bin), by its workgroup or, of up to
// 512 rows, by all CUs in two more launches (filter_count_kernel, filter_select_kernel<.., true>); the rest goes by a
// radix descent.  filter_bwd_kernel writes the gradient once and reads only the blocks that reach the border.
//
// What bounds it, and what it takes (us, kernels alone): the scan the memory where there are no sums (4096 rows of 151936 in bf16, half
// of them masked away: 129, 5.7 TB/s) or fp32 logits (384 rows of 151936: 46, 5.1 TB/s), the issue of its 10 operations of 64 bits per
// logit with sums of 16-bit ones (256 rows of 128257: 24, 2.7 TB/s); the selection a workgroup's chain of barriers (8 to 10 for a short
// nucleus, 20 for a long one), and where one CU passes over a row of very many candidates alone, its LDS atomics and arithmetic (36 for
// 50257 logits, 78 for 151936; 25 in parts, 8 for their launches where there is no such row); the gradient the memory (4096 rows of 151936: 222, 5.6 TB/s).
//
// Whole numbers come out, and the same ones whatever the launch: sums of weights are 64-bit floats in a fixed order over a row's
// chunks, or 64-bit integers (weights in units of 2^-fix, whose sums do not depend on the order in which threads add them).
#include <cfloat>
#include <type_traits>

#include "common.hpp"

namespace trlk {
namespace {

constexpr int kChunk = 2048;                 // logits of a wave of the scan
constexpr int kBlock = 64;                   // logits with a maximum of their own
constexpr int kBlocksPerChunk = kChunk / kBlock;
constexpr int kScanThreads = 256;
constexpr int kSelThreads = 512;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kBins = 4 * kSelThreads;       // of a step of the descent
constexpr int kBinBits = 11;
constexpr int kMaxCandidates = 4096;         // that are kept in LDS; rows with more read their blocks again in every step
constexpr int kList = 4096;                  // blocks over the bound that are listed; with more every block is looked at
constexpr int kPairs = 128;                  // candidates of which every pair is compared (256 rows with 100 of them 10.8 us, 13.1 by bins)
constexpr int kLine = 128;                   // bytes of a cache line
constexpr int kLongRows = 32;                // rows with very many candidates whose passes all CUs share
constexpr int kHalf = kChunk / 2;            // logits of a wave's step in these passes
constexpr int64_t kMaxVocab = int64_t(1) << 22;
// Temperatures up to it: over 2^100 logits further apart than the largest fp32 number could both count, and their distance is not one.  (Under it
// whatever is over 2^127 away from the maximum has no weight, and a bound that the filters set lies less than 2^111 under it.)
constexpr double kMaxTemperature = 0x1p100;
constexpr int64_t kMaxRows = (int64_t(1) << 32) / kSelThreads, kMaxUnits = (int64_t(1) << 32) / kWave - 8;

typedef unsigned long long u64;
#define TRLK_INLINE __attribute__((always_inline))
typedef u32x4 u32x4_u __attribute__((aligned(2)));  // a 16-byte vector at any element alignment

// ---- weights ---------------------------------------------------------------------------------------------------------
// 2^t for t <= 0 in 64 bits: 2^(t - n) on [-1/2, 1/2] by a polynomial of degree 9 that interpolates it at the Chebyshev points
// (relative error 4e-14), times 2^n.  -inf and everything under -1100 give 0.
__device__ __forceinline__ double exp2_f64(double t) {
    t = __builtin_fmax(t, -1100.0);
    const double n = __builtin_rint(t), f = t - n;
    double y = 1.0205905413765595e-07;
    y = __builtin_fma(y, f, 1.325964524488711e-06);
    y = __builtin_fma(y, f, 1.5252672924850737e-05);
    y = __builtin_fma(y, f, 0.0001540343375125101);
    y = __builtin_fma(y, f, 0.0013333558200794592);
    y = __builtin_fma(y, f, 0.009618129193934313);
    y = __builtin_fma(y, f, 0.05550410866465167);
    y = __builtin_fma(y, f, 0.2402265069564034);
    y = __builtin_fma(y, f, 0.6931471805599462);
    y = __builtin_fma(y, f, 1.0);  // (2^0 is 1 to the last bit: equal logits at the top have whole weights)
    return __builtin_amdgcn_ldexp(y, int(n));
}

// As above, of degree 11 (2e-17): for what a chunk's whole sum is multiplied by.
__device__ __forceinline__ double exp2_f64_exact(double t) {
    t = __builtin_fmax(t, -1100.0);
    const double n = __builtin_rint(t), f = t - n;
    double y = 4.4549605981865186e-10;
    y = __builtin_fma(y, f, 7.072585949269223e-09);
    y = __builtin_fma(y, f, 1.0178062445845774e-07);
    y = __builtin_fma(y, f, 1.321544258792169e-06);
    y = __builtin_fma(y, f, 1.525273382983612e-05);
    y = __builtin_fma(y, f, 0.0001540353044173605);
    y = __builtin_fma(y, f, 0.0013333558146416936);
    y = __builtin_fma(y, f, 0.009618129107606888);
    y = __builtin_fma(y, f, 0.0555041086648216);
    y = __builtin_fma(y, f, 0.24022650695910097);
    y = __builtin_fma(y, f, 0.6931471805599453);
    y = __builtin_fma(y, f, 1.0);
    return __builtin_amdgcn_ldexp(y, int(n));
}

// What a chunk's sum of weights is measured in.  Ordinarily 2^exponent, a whole number of at least max * c: x * c - exponent then needs one
// rounding, and its whole part takes one addition of a large number (`exp2_whole`).  Where
// max * c is too large for that, or neighbouring logits are so far apart that the clamp against underflow would not hold, the
// chunk's maximum itself, by subtraction.
struct ChunkUnit {
    double exponent;
    float x_min;  // logits under it count as it (2^-1000 at most)
    bool whole;
};
__device__ __forceinline__ ChunkUnit chunk_unit(float m, double c, double inv_c) {
    ChunkUnit u;
    u.exponent = m > -INFINITY ? __builtin_ceil(double(m) * c) : 0.0;
    u.x_min = float((u.exponent - 1000.0) * inv_c);
    const double t = __builtin_fma(double(u.x_min), c, -u.exponent);
    u.whole = u.exponent > -0x1p40 && u.exponent < 0x1p40 && t < -900.0 && t > -1020.0;
    return u;
}
// log2 of the unit of a chunk with maximum m, relative to a row's maximum
__device__ __forceinline__ double chunk_scale(float m, double c, double inv_c, double ref) {
    const ChunkUnit u = chunk_unit(m, c, inv_c);
    return m == -INFINITY ? -INFINITY : u.whole ? -__builtin_fma(ref, c, -u.exponent) : (double(m) - ref) * c;
}
// 2^(x * c - unit's exponent), 2^-1000 for an x of x_min: the number in 64ths comes from the low bits of x * c - exponent + 1.5 * 2^46, the
// root 2^(j / 64) of its low six bits from LDS, 2^f of the rest by 1 + f p(f) with p of degree 3 through the Chebyshev points of [-1/128, 1/128]
// (relative error 5e-15), and the whole powers go into the root's exponent.  10 operations of 64 bits, which are what bounds the scan, where a
// polynomial over [-1/2, 1/2] takes 15: 256 rows of 128257 in bf16 24 us instead of 27.
constexpr int kRoots = 64;
__device__ __forceinline__ double exp2_whole(float x, double c, double magic, const double* roots) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const double v = double(x), big = __builtin_fma(v, c, magic), f = __builtin_fma(v, c, magic - big);
    const uint32_t k = uint32_t(__builtin_bit_cast(uint64_t, big));
    u32x2 root = __builtin_bit_cast(u32x2, roots[k % kRoots]);
    root.y += k << 14;  // (the root has been stored without the part of it that is below the exponent)
    const double r = __builtin_bit_cast(double, root);
    double p = 0.009618138509201629;
    p = __builtin_fma(p, f, 0.05550419004645178);
    p = __builtin_fma(p, f, 0.24022650695902897);
    p = __builtin_fma(p, f, 0.6931471805593244);
    return __builtin_fma(r * f, p, r);
}
__device__ __forceinline__ double stored_root(int j) {
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, exp2(double(j) / kRoots)) - (uint64_t(j) << 46));
}

// maximum that lets a NaN through
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// v of the lane that differs in one bit of its number (1, 2), or that mirrors it in 8 or 16
template <int CTRL>
__device__ __forceinline__ float moved_f32(float v) {
    return __uint_as_float(uint32_t(__builtin_amdgcn_mov_dpp(int(__float_as_uint(v)), CTRL, 0xf, 0xf, true)));
}
// maximum over groups of LANES neighbouring lanes (8 or 16)
template <int LANES>
__device__ __forceinline__ float group_max_nan(float v) {
    v = max_nan(v, moved_f32<0xb1>(v));
    v = max_nan(v, moved_f32<0x4e>(v));
    v = max_nan(v, moved_f32<0x141>(v));
    if constexpr (LANES == 16) v = max_nan(v, moved_f32<0x140>(v));
    return v;
}
__device__ __forceinline__ float wave_max_nan(float v) {
    v = group_max_nan<16>(v);
    v = max_nan(v, __shfl_xor(v, 16));
    return max_nan(v, __shfl_xor(v, 32));
}

// A 64-bit value from the lane that the data-parallel primitive names, 0 where there is none.
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V moved(V v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b)), CTRL, ROWS, 0xf, false));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), CTRL, ROWS, 0xf, false));
    return __builtin_bit_cast(V, uint64_t(hi) << 32 | lo);
}
// Sums over the lanes up to each one: shifts within rows of 16 lanes, then the last lane of row 0 (2) to row 1 (3), that of row 1 to
// rows 2 and 3.  A fifth of the time that six shuffles through LDS take.
template <typename V>
__device__ __forceinline__ V wave_inclusive(V v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v) {
    const auto add = [&](auto moved_of) TRLK_INLINE { v += uint32_t(moved_of(int(v))); };
    add([](int x) TRLK_INLINE { return __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false); });
    add([](int x) TRLK_INLINE { return __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false); });
    add([](int x) TRLK_INLINE { return __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false); });
    add([](int x) TRLK_INLINE { return __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false); });
    add([](int x) TRLK_INLINE { return __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false); });
    add([](int x) TRLK_INLINE { return __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false); });
    return v;
}
// A place for each of a wave's items in a list in LDS: `count` of this lane, all lanes in it.
__device__ __forceinline__ uint32_t reserve(uint32_t* size, uint32_t count) {
    const uint32_t inc = wave_inclusive(count), total = uint32_t(__builtin_amdgcn_readlane(int(inc), kWave - 1));
    if (total == 0) return 0;
    uint32_t base = 0;
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) base = atomicAdd(size, total);
    return uint32_t(__builtin_amdgcn_readlane(int(base), kWave - 1)) + inc - count;
}

// Unsigned numbers in the order of the values (16 bits for 16-bit types).  -0 comes right before +0: they are different keys of
// equal values, so it is read as +0.
template <int DT>
struct Key {
    static constexpr bool k16 = DT != TRLK_F32;
    typedef typename Elem<DT>::type raw;
    static __device__ __forceinline__ uint32_t of(raw r) {
        if constexpr (k16) {
            const uint32_t u = r == 0x8000u ? 0u : r;
            return u & 0x8000u ? 0xffffu - u : u | 0x8000u;
        } else {
            const uint32_t b = __float_as_uint(r), u = b == 0x80000000u ? 0u : b;
            return u & 0x80000000u ? ~u : u | 0x80000000u;
        }
    }
    static __device__ __forceinline__ raw value(uint32_t k) {
        if constexpr (k16)
            return raw(k & 0x8000u ? k & 0x7fffu : 0xffffu - k);
        else
            return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
    }
    static __device__ __forceinline__ float to_float(uint32_t k) { return Elem<DT>::to_float(value(k)); }
    static __device__ __forceinline__ uint32_t of_float(float x) {  // (x is a value of the type)
        raw r;
        if constexpr (k16)
            Elem<DT>::store1(&r, x);
        else
            r = x;
        return of(r);
    }
};

// ---- a row's settings ------------------------------------------------------------------------------------------------
struct Filters {
    double temperature, top_p, min_p;
    int64_t top_k;
    const float *d_temperature, *d_top_p, *d_min_p;  // a value for each row, or null: the number above
    const int32_t* d_top_k;
    double c, inv_c;  // log2(e) / temperature and its inverse (a division of 64 bits costs a wave as much as two of its logits)
};
struct RowFilter {
    double c, inv_c;  // log2(e) / T and T / log2(e)
    double top_p;     // 0: not in force
    double min_p;     // 0: not in force
    uint32_t top_k;   // 0: not in force
    bool ok;
};
__device__ __forceinline__ RowFilter row_filter(const Filters& f, int64_t row, int64_t vocab) {
    double T = f.d_temperature ? double(f.d_temperature[row]) : f.temperature;
    const double p = f.d_top_p ? double(f.d_top_p[row]) : f.top_p;
    const double q = f.d_min_p ? double(f.d_min_p[row]) : f.min_p;
    int64_t k = f.d_top_k ? int64_t(f.d_top_k[row]) : f.top_k;
    RowFilter r;
    r.ok = T >= 0.0 && T <= kMaxTemperature && p == p && q == q;
    if (T == 0.0) {
        T = 1.0;
        k = 1;
    }
    r.c = f.d_temperature ? 1.4426950408889634074 / T : f.c;
    r.inv_c = f.d_temperature ? 0.69314718055994530942 * T : f.inv_c;
    r.ok = r.ok && r.c < INFINITY;
    r.top_k = k > 0 && k < vocab ? uint32_t(k) : 0u;
    r.top_p = p >= 1.0 ? 0.0 : __builtin_fmax(p, 1e-300);  // (0 or less keeps the first token, as the smallest positive number does)
    r.min_p = q <= 0.0 ? 0.0 : __builtin_fmin(q, 1.0);
    return r;
}

struct RowView {
    const void* logits;
    int64_t rows_per_seq, vocab, seq_stride, row_stride;
    template <int DT>
    __device__ __forceinline__ const typename Elem<DT>::type* row(uint32_t r) const {  // (rows are fewer than 2^23)
        const uint32_t b = r / uint32_t(rows_per_seq), t = r - b * uint32_t(rows_per_seq);
        return static_cast<const typename Elem<DT>::type*>(logits) + int64_t(b) * seq_stride + int64_t(t) * row_stride;
    }
};

// ---- rows with very many candidates ------------------------------------------------------------------------------------
// What the selection leaves of such a row for the two launches behind it, which pass over it in parts.
struct alignas(64) LongRow {
    double sum;      // of the row's weights
    u64 mass;        // before the bins that have the border
    float m, x_low;  // the row's maximum, and what no candidate lies under
    uint32_t row, n_zone, min_key, done;
    __device__ u64* bins() { return reinterpret_cast<u64*>(this + 1); }
    __device__ u64* zone() { return bins() + kBins; }
};
constexpr size_t kLongRowBytes = sizeof(LongRow) + sizeof(u64) * (kBins + kMaxCandidates);
struct LongRows {
    uint32_t* count;  // null: no row can be one.  More rows than there are slots are passed over by their own workgroups
    char* slots;
    uint32_t n_slots;
    int32_t parts;    // workgroups that share a row's pass, one half chunk to a wave
    __device__ LongRow* at(uint32_t i) const { return reinterpret_cast<LongRow*>(slots + i * kLongRowBytes); }
    __device__ bool has(uint32_t i) const { return i < *count; }
};

// ---- scan ------------------------------------------------------------------------------------------------------------
struct ScanArgs {
    RowView x;
    int64_t rows;
    int32_t chunks;
    Filters f;
    const uint8_t* row_mask;
    double* chunk_sum;  // [rows, chunks] or null
    float* chunk_max;   // [rows, chunks]
    void* block_max;    // [rows, chunks * kBlocksPerChunk] in the logits' type, or null
    uint32_t* long_count;  // set to 0, or null
};

// NV vectors of a lane: vector i holds the logits (i * 64 + lane) * EPV on of those at p.  What lies behind the n there are is -inf.
template <int DT, int NV>
__device__ __forceinline__ void load_vectors(const typename Elem<DT>::type* p, int64_t n, int lane, float (&x)[NV * Elem<DT>::EPV]) {
    constexpr int EPV = Elem<DT>::EPV;
    if (n >= NV * kWave * EPV) {
        u32x4 q[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = *reinterpret_cast<const u32x4_u*>(p + (i * kWave + lane) * EPV);
#pragma unroll
        for (int i = 0; i < NV; ++i) Elem<DT>::unpack(q[i], x + i * EPV);
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * kWave + lane) * EPV;
        if (at + EPV <= n) {
            const u32x4 q = *reinterpret_cast<const u32x4_u*>(p + at);
            Elem<DT>::unpack(q, x + i * EPV);
        } else {
#pragma unroll
            for (int e = 0; e < EPV; ++e) x[i * EPV + e] = at + e < n ? Elem<DT>::load1(p + at + e) : -INFINITY;
        }
    }
}

template <int DT, int NV>
__device__ __forceinline__ void load_raw(const typename Elem<DT>::type* p, int64_t n, int lane, u32x4 (&q)[NV]) {
    constexpr int EPV = Elem<DT>::EPV;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * kWave + lane) * EPV;
        if (at + EPV <= n) {
            q[i] = *reinterpret_cast<const u32x4_u*>(p + at);
        } else {
            float x[EPV];
#pragma unroll
            for (int e = 0; e < EPV; ++e) x[e] = at + e < n ? Elem<DT>::load1(p + at + e) : -INFINITY;
            q[i] = Elem<DT>::pack(x);
        }
    }
}

template <int DT, bool SUMS, bool BLOCKS>
__global__ __launch_bounds__(kScanThreads, 8) void filter_scan_kernel(ScanArgs a) {
    typedef typename Elem<DT>::type T;
    constexpr int EPV = Elem<DT>::EPV, NV = kChunk / (kWave * EPV), LPB = kBlock / EPV;  // LPB: lanes of a block
    __shared__ double roots[SUMS ? kRoots : 1];
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.long_count) *a.long_count = 0;
    if constexpr (SUMS) {
        if (threadIdx.x < kRoots) roots[threadIdx.x] = stored_root(int(threadIdx.x));
        __syncthreads();
    }
    const int lane = threadIdx.x & (kWave - 1);
    const uint32_t at_unit = __builtin_amdgcn_readfirstlane(int(blockIdx.x * (kScanThreads / kWave) + threadIdx.x / kWave));
    const uint32_t at_row = at_unit / uint32_t(a.chunks);  // (units are fewer than 2^26)
    const int64_t unit = at_unit, row = at_row;
    if (row >= a.rows) return;
    const int chunk = int(at_unit - at_row * uint32_t(a.chunks));
    if (a.row_mask && a.row_mask[row] == 0) return;
    const T* p = a.x.row<DT>(uint32_t(row)) + int64_t(chunk) * kChunk;
    float x[NV * EPV];
    load_vectors<DT, NV>(p, a.x.vocab - int64_t(chunk) * kChunk, lane, x);
    float m = -INFINITY, mine = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float v = x[i * EPV];
#pragma unroll
        for (int e = 1; e < EPV; ++e) v = max_nan(v, x[i * EPV + e]);
        if constexpr (BLOCKS) {
            v = group_max_nan<LPB>(v);
            if ((lane & (LPB - 1)) == i) mine = v;
        }
        m = max_nan(m, v);
    }
    if constexpr (BLOCKS) {  // lane l has the maximum of vector l % LPB, block l / LPB
        const int i = lane & (LPB - 1);
        T* out = static_cast<T*>(a.block_max) + unit * kBlocksPerChunk;
        if (i < NV) Elem<DT>::store1(out + i * (kWave / LPB) + lane / LPB, mine);
    }
    m = wave_max_nan(m);
    if constexpr (SUMS) {
        const RowFilter f = row_filter(a.f, row, a.x.vocab);
        const double c = f.c;
        const ChunkUnit in = chunk_unit(m, c, f.inv_c);
        double s = 0.0;
        if (in.whole) {
            const double magic = 0x1.8p46 - in.exponent;
#pragma unroll
            for (int j = 0; j < NV * EPV; ++j) s += exp2_whole(max_nan(x[j], in.x_min), c, magic, roots);
        } else {
#pragma unroll
            for (int j = 0; j < NV * EPV; ++j) s += exp2_f64((double(x[j]) - double(m)) * c);
        }
        s = wave_inclusive(s);
        if (lane == kWave - 1) a.chunk_sum[unit] = s;
    }
    if (lane == 0) a.chunk_max[unit] = m;
}

// ---- select ----------------------------------------------------------------------------------------------------------
struct SelectArgs {
    RowView x;
    int64_t rows;
    int32_t chunks, fix;
    Filters f;
    const uint8_t* row_mask;
    double* chunk_sum;  // (a row with very many candidates puts the kept weights of its chunks there)
    const float* chunk_max;
    const void* block_max;
    int32_t has_blocks, has_sums;  // what the scan has left
    const void* uniform;  // sample: fp32 or fp64 [rows]
    int32_t uniform_f64;
    int64_t fill_id;
    int64_t* out_ids;
    const int64_t* index;  // score: [rows]
    float* out_state;      // score: [rows, 4]: border value, border index (bits), maximum, log2 of the kept mass in units of its weight
    float* out_logp;
    int32_t* error_flag;
    LongRows longs;
};

// A place for one number of each wave.  Two neighbouring block-wide sums take different ones, so that a barrier lies between a
// place's readers and its next writers.
union WaveSlots {
    u64 u[kSelWaves];
    double f[kSelWaves];
};
__device__ __forceinline__ u64& slot_of(WaveSlots& s, int i, u64) { return s.u[i]; }
__device__ __forceinline__ double& slot_of(WaveSlots& s, int i, double) { return s.f[i]; }

template <int CANDIDATES>
struct SelectShared {
    u64 bins[kBins];
    u64 order[CANDIDATES];  // of the candidates: key above, ~index below, larger is earlier
    u64 weight[kPairs], zone[kPairs];
    uint16_t list[kList];
    WaveSlots slots[4];
    float wave_f[kSelWaves];
    int hit[2][kSelWaves], tail[2][kSelWaves];
    double prefix[kSelWaves];
    u64 before;
    uint32_t bin, n_list, n_cand, n_zone, min_key, low_key, border, border_index;
};

// Sums over the threads before this one (returned) and up to it (`upto`), and over all.  What one thread's `upto` is, is the next
// one's exclusive sum to the last bit.  Contains one barrier.
template <typename V>
__device__ __forceinline__ V block_scan(V v, WaveSlots& slots, V& upto, V& total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const V inc = wave_inclusive(v);
    V exc = __shfl_up(inc, 1);
    if (lane == 0) exc = 0;
    if (lane == kWave - 1) slot_of(slots, wave, v) = inc;
    __syncthreads();
    V base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
        if (w == wave) base = all;
        all += slot_of(slots, w, v);
    }
    total = all;
    upto = base + inc;
    return base + exc;
}
__device__ __forceinline__ u64 block_total(u64 v, WaveSlots& slots) {
    const u64 inc = wave_inclusive(v);
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) slots.u[threadIdx.x / kWave] = inc;
    __syncthreads();
    u64 r = 0;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) r += slots.u[w];
    return r;
}

// The bin up to which the values of bins [0, n) and `before` reach a target first, and in `before` what lies before it; false if
// all of them do not.  The target comes from the sum of all bins.  The bins are complete and the barrier behind them passed; s.bin
// is ~0.  Contains two barriers.
template <typename Shared, typename Target>
__device__ __forceinline__ bool crossing_of(Shared& s, int n, Target target_of, uint32_t& bin, u64& before) {
    u64 v[4], sum = 0, upto, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = 4 * threadIdx.x + j;
        v[j] = i < n ? s.bins[i] : 0;
        sum += v[j];
    }
    u64 at = before + block_scan(sum, s.slots[0], upto, total);
    const u64 target = target_of(total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (at < target && at + v[j] >= target) {  // (one bin of one thread)
            s.bin = 4 * threadIdx.x + j;
            s.before = at;
        }
        at += v[j];
    }
    __syncthreads();
    bin = s.bin;
    if (bin == ~0u) return false;
    before = s.before;
    return true;
}
template <typename Shared>
__device__ __forceinline__ bool crossing(Shared& s, int n, u64 target, uint32_t& bin, u64& before) {
    return crossing_of(s, n, [&](u64) TRLK_INLINE { return target; }, bin, before);
}
// all bins 0 and no crossing yet, behind a barrier
template <typename Shared>
__device__ __forceinline__ void clear_bins(Shared& s, int n) {
    for (int i = threadIdx.x; i < n; i += kSelThreads) s.bins[i] = 0;
    __syncthreads();
    if (threadIdx.x == 0) s.bin = ~0u;  // (everyone has read the last one, and two barriers lie before the next is written)
}

// The first n <= kPairs entries of an order and their weights in LDS, each compared with every other one: what comes before it in the
// order (of its bits under `mask`; larger is earlier), how many and of which weight.  `parts` neighbouring lanes have an entry
// together and a part of the others each; the first of them goes on with it.  Up to np entries behind the n are overwritten;
// contains one barrier, after which both arrays may be read.
struct Ranked {
    u64 order, weight, before;
    uint32_t rank;
    bool real;
};
__device__ __forceinline__ Ranked rank_pairs(u64* order, u64* weight, int n, u64 mask) {
    const int tid = threadIdx.x, lp = n <= 64 ? 3 : 2, parts = 1 << lp, np = kSelThreads >> lp, len = np >> lp;
    const int i = tid >> lp, part = tid & (parts - 1);
    if (tid >= n && tid < np) order[tid] = weight[tid] = 0;
    __syncthreads();
    Ranked r;
    r.order = order[i];
    r.weight = weight[i];
    r.real = i < n && part == 0;
    const u64 me = r.order & mask;
    u64 before = 0, rank = 0;
    for (int j0 = 0; j0 < len; j0 += 8) {
        u64 o[8], w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            o[j] = order[(j0 + j) * parts + part];
            w[j] = weight[(j0 + j) * parts + part];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool earlier = (o[j] & mask) > me;
            before += earlier ? w[j] : 0;
            rank += earlier ? 1 : 0;
        }
    }
    const auto over_parts = [&](u64 v) TRLK_INLINE {
        v += moved<0xb1, 0xf>(v);                  // the neighbour
        v += moved<0x4e, 0xf>(v);                  // the other pair of four
        if (parts > 4) v += moved<0x141, 0xf>(v);  // the mirrored lane of eight
        return v;
    };
    r.before = over_parts(before);
    r.rank = uint32_t(over_parts(rank));
    return r;
}
constexpr u64 kByOrder = ~u64(0), kByIndex = 0xffffffffu;

// The smallest position in [lo, hi] up to which `before` and the values reach `target`, and in `before` what lies before it.
// `each(f)` calls f(position, value) for this thread's share of the items.  False if all of them do not reach it.
template <typename Shared, typename Each>
__device__ __forceinline__ bool descend(Shared& s, Each each, uint32_t lo, uint32_t hi, u64 target, uint32_t& position, u64& before) {
    for (;;) {
        const uint32_t span = hi - lo;
        const int bits = span ? 32 - __builtin_clz(span) : 0, shift = bits > kBinBits ? bits - kBinBits : 0;
        const int n = int(span >> shift) + 1;
        clear_bins(s, n);
        each([&](uint32_t at, u64 value) {
            if (at >= lo && at <= hi && value) atomicAdd(&s.bins[(at - lo) >> shift], value);
        });
        __syncthreads();
        uint32_t bin;
        if (!crossing(s, n, target, bin, before)) return false;
        lo += bin << shift;
        position = lo;
        if (shift == 0) return true;
        const uint32_t last = lo + ((1u << shift) - 1u);
        hi = last < hi ? last : hi;
    }
}

// Distance from the maximum in bins of 1/128 of itself: 0 for less than 2^-8, then 128 bins for each power of two.  Monotone, and it
// depends neither on where a row's logits lie nor on the temperature.
__device__ __forceinline__ int distance_bin(float m, float x) {
    const int b = int(__float_as_uint(m - x) >> 16) - (119 << 7);
    return b > 0 ? b : 0;
}
constexpr int kEveryBin = 1 << 30;

// Bins of a row with very many candidates: the logits down to x_low, and of each bin the count and the sum of the places in it, in 256ths.
__device__ __forceinline__ float bins_per_logit(float m, float x_low) { return float(kBins - 1) / fmaxf(m - x_low, 1e-30f); }
template <int N>
__device__ __forceinline__ void count_in_bins(const float (&v)[N], float m, float scale, u64* bins) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const uint32_t t = uint32_t((m - v[e]) * (256.f * scale));  // (infinity is the largest number)
        if (t < 256u * kBins) atomicAdd(&bins[t / 256u], u64(1) << 32 | t % 256u);
    }
}

// `owner` of the smallest thread number, and if there is none of the largest with `some`: its number, the same for all threads
template <typename Shared>
__device__ __forceinline__ int first_thread(Shared& s, int which, bool owner, bool some) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const u64 a = __ballot(owner), b = __ballot(some);
    if (lane == 0) {
        s.hit[which][wave] = a ? wave * kWave + __builtin_ctzll(a) : -1;
        s.tail[which][wave] = b ? wave * kWave + 63 - __builtin_clzll(b) : -1;
    }
    __syncthreads();
    int r = -1;
#pragma unroll
    for (int w = kSelWaves - 1; w >= 0; --w)
        if (s.hit[which][w] >= 0) r = s.hit[which][w];
    if (r >= 0) return r;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w)
        if (s.tail[which][w] >= 0) r = s.tail[which][w];
    return r;
}

// LONG: rows may have no top-k, and so any number of tokens, or no filter at all.  Without, three workgroups fit into a CU instead of two:
// 4096 rows of 151936 with top-k and top-p 39 us instead of 50.
// SECOND: a part of the second pass over one of the rows that the selection has left; the workgroup that is through last goes on alone.
template <int DT, bool SCORE, bool LONG, bool SECOND = false>
__global__ __launch_bounds__(kSelThreads, LONG ? 4 : 6) void filter_select_kernel(SelectArgs a) {
    typedef typename Elem<DT>::type T;
    typedef Key<DT> K;
    constexpr int EPV = Elem<DT>::EPV, PER = kChunk / kSelThreads;
    constexpr int NV = kChunk / (kWave * EPV);
    constexpr int kKeep = sizeof(T) == 4 ? 2 : 1;  // vectors of block maxima that a thread holds: 4096 blocks
    constexpr int kCandidates = LONG ? kMaxCandidates : kMaxCandidates / 2;
    __shared__ SelectShared<kCandidates> s;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    LongRow* const left = SECOND ? a.longs.at(blockIdx.y) : nullptr;
    if (SECOND && !a.longs.has(blockIdx.y)) return;
    const int64_t row = SECOND ? left->row : blockIdx.x, V = a.x.vocab;
    // what a row without a token, or without a distribution, returns
    const auto nothing = [&](int64_t id, float logp) TRLK_INLINE {
        if (tid != 0) return;
        if constexpr (SCORE) {
            a.out_state[row * 4] = INFINITY;
            a.out_state[row * 4 + 1] = a.out_state[row * 4 + 2] = a.out_state[row * 4 + 3] = 0.f;
        } else {
            a.out_ids[row] = id;
        }
        a.out_logp[row] = logp;
    };
    if (!SECOND && a.row_mask && a.row_mask[row] == 0) return nothing(a.fill_id, 0.f);
    // (what every row needs is on its way before the row's settings are known)
    const float* cmax = a.chunk_max + row * a.chunks;
    double* csum = a.chunk_sum + row * a.chunks;
    const int n_blocks = a.chunks * kBlocksPerChunk, n_vec = n_blocks / EPV;  // (blocks behind the row's end are -inf)
    const u32x4* bmax = reinterpret_cast<const u32x4*>(static_cast<const T*>(a.block_max) + row * n_blocks);
    u32x4 held[kKeep] = {};
    if (!SECOND && a.has_blocks) {
#pragma unroll
        for (int j = 0; j < kKeep; ++j)
            if (tid + j * kSelThreads < n_vec) held[j] = bmax[tid + j * kSelThreads];
    }
    const int per = (a.chunks + kSelThreads - 1) / kSelThreads, first = tid * per, last = first + per < a.chunks ? first + per : a.chunks;
    double sum0 = 0.0;  // this thread's first chunk
    float max0 = -INFINITY;
    if (LONG && !SECOND && a.has_sums && first < last) {
        sum0 = csum[first];
        max0 = cmax[first];
    }
    const RowFilter f = row_filter(a.f, row, V);
    const bool filtered = !LONG || SECOND || f.top_k || f.top_p > 0.0 || f.min_p > 0.0;
    const bool with_sum = LONG && (!filtered || (f.top_p > 0.0 && !f.top_k));
    const T* x = a.x.row<DT>(uint32_t(row));

    // the row's maximum: of its blocks, or of its chunks where there are no blocks
    float m = -INFINITY;
    if (SECOND) {
        m = left->m;
    } else if (filtered) {
#pragma unroll
        for (int j = 0; j < kKeep; ++j) {
            float v[EPV];
            Elem<DT>::unpack(held[j], v);
            if (tid + j * kSelThreads < n_vec) {
#pragma unroll
                for (int e = 0; e < EPV; ++e) m = max_nan(m, v[e]);
            }
        }
        for (int i = tid + kKeep * kSelThreads; i < n_vec; i += kSelThreads) {
            float v[EPV];
            Elem<DT>::unpack(bmax[i], v);
#pragma unroll
            for (int e = 0; e < EPV; ++e) m = max_nan(m, v[e]);
        }
    } else {
        for (int i = tid; i < a.chunks; i += kSelThreads) m = max_nan(m, cmax[i]);
    }
    int64_t token = 0;
    bool token_ok = true;
    T token_raw = 0;
    if constexpr (SCORE) {
        token = a.index[row];
        token_ok = token >= 0 && token < V;
        if (token_ok) token_raw = x[token];
        if (!token_ok && tid == 0 && a.error_flag) atomicOr(a.error_flag, TRLK_FLAG_INDEX_OUT_OF_RANGE);
    }
    double u = 0.0;
    if constexpr (!SCORE) {
        u = a.uniform_f64 ? static_cast<const double*>(a.uniform)[row] : double(static_cast<const float*>(a.uniform)[row]);
        u = u > 0.0 ? u : 0.0;  // (and NaN)
    }
    if (filtered)
        for (int i = tid; i < kBins; i += kSelThreads) s.bins[i] = 0;
    m = wave_max_nan(m);
    if (lane == 0) s.wave_f[wave] = m;
    if (tid == 0) {
        s.n_list = s.n_cand = s.n_zone = 0;
        s.min_key = s.low_key = s.bin = ~0u;
    }
    __syncthreads();
    m = s.wave_f[0];
#pragma unroll
    for (int w = 1; w < kSelWaves; ++w) m = max_nan(m, s.wave_f[w]);
    if (!f.ok || !(m < INFINITY) || m == -INFINITY) {
        if (tid == 0 && a.error_flag) atomicOr(a.error_flag, TRLK_FLAG_NO_DISTRIBUTION);
        return nothing(-1, NAN);
    }
    const double c = f.c, ref = double(m), unit = __builtin_amdgcn_ldexp(1.0, a.fix);
    const auto weight = [&](float v) TRLK_INLINE { return exp2_f64((double(v) - ref) * c); };
    const auto chunk_weight = [&](double sum, float chunk_m) TRLK_INLINE { return sum * exp2_f64_exact(chunk_scale(chunk_m, c, f.inv_c, ref)); };
    // w <= 1 in units of 2^-fix, rounded to the nearest: the low bits of a sum with 1.5 * 2^52 (fix is at most 50)
    const auto fixed = [&](double w) TRLK_INLINE { return __builtin_bit_cast(u64, __builtin_fma(w, unit, 0x1.8p52)) - __builtin_bit_cast(u64, 0x1.8p52); };
    const auto log2_of = [&](u64 W) TRLK_INLINE { return log2(double(W)) - a.fix; };
    const auto drawn = [&](int64_t id, float v, double log2_mass) TRLK_INLINE {  // one thread
        a.out_ids[row] = id;
        a.out_logp[row] = float(((double(v) - ref) * c - log2_mass) * 0.69314718055994530942);
    };
    const auto scored = [&](uint32_t border, uint32_t border_index, auto mass) TRLK_INLINE {  // all threads
        if (tid != 0) return;
        const double log2_mass = mass();
        float logp = NAN;
        bool inside = false;
        if (token_ok) {
            const float v = Elem<DT>::to_float(token_raw);
            const uint32_t k = K::of(token_raw);
            inside = v > -INFINITY && (!filtered || k > border || (k == border && uint32_t(token) <= border_index));
            logp = inside ? float(((double(v) - ref) * c - log2_mass) * 0.69314718055994530942) : -INFINITY;
        }
        float* st = a.out_state + row * 4;
        st[0] = !inside ? INFINITY : filtered ? K::to_float(border) : -INFINITY;  // (no gradient reaches a row whose token lies outside)
        st[1] = __uint_as_float(border_index);
        st[2] = m;
        st[3] = float(log2_mass);
        a.out_logp[row] = logp;
    };

    // the row's sum of weights, and this thread's chunks' place in it
    double S = 0.0, mine = 0.0, base = 0.0, upto = 0.0;
    if (SECOND) {
        S = left->sum;
    } else if (with_sum) {
        if (first < last) mine = chunk_weight(sum0, max0);
        for (int i = first + 1; i < last; ++i) mine += chunk_weight(csum[i], cmax[i]);
        base = block_scan(mine, s.slots[1], upto, S);
    }
    // ---- no filter: the chunk, then the token in it
    if (LONG && !filtered) {
        if constexpr (SCORE) {
            return scored(0, ~0u, [&]() TRLK_INLINE { return log2(S); });
        } else {
            // (u * S can round up to the whole sum, and the last bits of a scan are not monotone: the first thread whose sum passes it,
            // and that has something, or the last one that has)
            const double target = u * S;
            const int owner = first_thread(s, 0, mine > 0.0 && upto > target, mine > 0.0);
            if (tid == owner) {
                double at = base, v = chunk_weight(sum0, max0);
                int chunk = first, some = v > 0.0 ? first : -1;
                double some_at = at;
                for (;;) {
                    if (v > 0.0) {
                        some = chunk;
                        some_at = at;
                        if (at + v > target) break;
                    }
                    at += v;
                    if (++chunk >= last) break;
                    v = chunk_weight(csum[chunk], cmax[chunk]);
                }
                s.border = uint32_t(some);
                s.prefix[0] = some_at;
            }
            __syncthreads();
            const int chunk = int(s.border);
            const double prefix = s.prefix[0];
            double w[PER], sum = 0.0, up, all;
            float v[PER];
            const int64_t e0 = int64_t(chunk) * kChunk + tid * PER;
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = e0 + j < V ? Elem<DT>::load1(x + e0 + j) : -INFINITY;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                w[j] = weight(v[j]);
                sum += w[j];
            }
            double run = prefix + block_scan(sum, s.slots[2], up, all);
            const int at = first_thread(s, 1, sum > 0.0 && prefix + up > target, sum > 0.0);
            if (tid == at) {
                int some = 0;
                float vs = v[0];
                bool past = false;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    run += w[j];
                    if (w[j] > 0.0 && !past) {
                        some = j;
                        vs = v[j];
                        past = run > target;
                    }
                }
                drawn(e0 + some, vs, log2(S));
            }
            return;
        }
    }

    // ---- a bound under the border, in bins of the distance from the maximum
    const auto key_of = [&](u64 order) TRLK_INLINE { return uint32_t(order >> 32); };
    const auto index_of = [&](u64 order) TRLK_INLINE { return ~uint32_t(order); };
    const auto order_of = [&](float v, uint32_t e) TRLK_INLINE { return u64(K::of_float(v)) << 32 | uint32_t(~e); };
    const auto key_weight = [&](uint32_t k) TRLK_INLINE { return weight(K::to_float(k)); };
    const auto each_max = [&](auto g) TRLK_INLINE {  // g(vector, its values), all lanes of a wave together; there may be none (-inf)
        const auto vec = [&](int i, u32x4 q) TRLK_INLINE {
            float v[EPV];
            Elem<DT>::unpack(q, v);
#pragma unroll
            for (int e = 0; e < EPV; ++e) v[e] = i < n_vec ? v[e] : -INFINITY;
            g(i, v);
        };
#pragma unroll
        for (int j = 0; j < kKeep; ++j) vec(tid + j * kSelThreads, held[j]);
        for (int i = kKeep * kSelThreads; i < n_vec; i += kSelThreads) vec(i + tid, i + tid < n_vec ? bmax[i + tid] : u32x4{0, 0, 0, 0});
    };
    // weights in fp32, in units of 2^-31 of the row's sum (off by 1e-5 at most, and half a unit): they narrow down, nothing is decided by them
    const float cf = float(c), l2 = 31.f - __builtin_amdgcn_logf(float(S));
    const auto about = [&](float v) TRLK_INLINE { return uint32_t(fast_exp2(fmaf(v - m, cf, l2)) + 0.5f); };
    const auto add_low = [&](int bin, uint32_t v) TRLK_INLINE { atomicAdd(reinterpret_cast<uint32_t*>(&s.bins[bin]), v); };  // (sums under 2^32)
    const u64 mass_target = [&]() TRLK_INLINE {  // of top-p without top-k
        // (S is off by up to 1.1e-14 of itself: 5e-15 in the powers, the rest in the sums.  A border that lies closer counts as reached: of 8 equal
        // logits top_p = 0.5 keeps 4, also where S is 8 and a few last bits)
        const double t = __builtin_ceil(f.top_p * S * (1.0 - 1.2e-14) * unit);
        return t < 1.0 ? u64(1) : u64(int64_t(t));
    }();
    int bound = kEveryBin;
    float x_low = -INFINITY;  // no candidate lies under it
    if (SECOND) {
        x_low = left->x_low;
    } else {
        const bool by_count = f.top_k != 0, by_mass = !by_count && f.top_p > 0.0;
        if (by_count || by_mass) {
            each_max([&](int, const float(&v)[EPV]) TRLK_INLINE {
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    const int d = distance_bin(m, v[e]);
                    if (d < kBins) add_low(d, by_count ? 1u : about(v[e]));
                }
            });
            __syncthreads();
            uint32_t bin;
            u64 before = 0;
            if (crossing(s, kBins, by_count ? u64(f.top_k) : u64(f.top_p * 0x1p31 * (1.0 + 1e-5)) + n_blocks, bin, before)) bound = int(bin);
        }
        if (by_mass) {  // all tokens of less than (1 - top_p) / V of the mass together have less than 1 - top_p of it
            x_low = float(ref + log2((1.0 - f.top_p) * S / double(V) * (1.0 - 1e-9)) / c);
            x_low -= 1e-6f * fabsf(x_low) + 1e-30f;
        }
        if (f.min_p > 0.0 && !(f.top_k && f.top_p > 0.0)) {  // (top-p of top-k counts what min-p takes away)
            float b = float(ref + log2(f.min_p) / c);
            b -= 1e-6f * fabsf(b) + 1e-30f;
            x_low = fmaxf(x_low, b);
        }
        if (x_low > -INFINITY) {
            const int d = distance_bin(m, x_low);
            bound = d < bound ? d : bound;
        }
    }
    // (the same bin or a nearer one: a distance of at most the largest number of that bin)
    const float reach = bound < kEveryBin ? __uint_as_float((uint32_t(bound + (119 << 7) + 1) << 16) - 1u) : INFINITY;
    const auto in_bound = [&](float v) TRLK_INLINE { return v > -INFINITY && m - v <= reach; };

    // ---- blocks that reach the bound, and the candidates in them
    if (!SECOND) each_max([&](int i, const float(&v)[EPV]) TRLK_INLINE {
        uint32_t in = 0;
#pragma unroll
        for (int e = 0; e < EPV; ++e) in |= in_bound(v[e]) ? 1u << e : 0u;
        uint32_t to = reserve(&s.n_list, __popc(in));
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
            if (in >> e & 1u) {
                if (to < kList) s.list[to] = uint16_t(i * EPV + e);
                ++to;
            }
        }
    });
    __syncthreads();
    const bool listed = !SECOND && s.n_list <= kList;
    const int n_visit = listed ? int(s.n_list) : n_blocks;
    // the logits of those blocks, EPV blocks to a load of a wave and U loads together: g(vectors, indices of their first logits)
    constexpr int U = LONG ? 4 : 2;
    const auto blocks_raw = [&](auto g) TRLK_INLINE {
        constexpr int LPB = kBlock / EPV;
        for (int j0 = wave * EPV; j0 < n_visit; j0 += U * kSelWaves * EPV) {
            u32x4 raw[U];
            int e[U];
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int j = j0 + q * kSelWaves * EPV + lane / LPB;
                e[q] = j < n_visit ? (listed ? int(s.list[j]) : j) * kBlock + (lane & (LPB - 1)) * EPV : int(V);
                if (e[q] + EPV <= int(V)) {
                    raw[q] = *reinterpret_cast<const u32x4_u*>(x + e[q]);
                } else {
                    float v[EPV];
#pragma unroll
                    for (int k = 0; k < EPV; ++k) v[k] = e[q] + k < int(V) ? Elem<DT>::load1(x + e[q] + k) : -INFINITY;
                    raw[q] = Elem<DT>::pack(v);
                }
            }
            g(raw, e);
        }
    };
    const auto blocks_pass = [&](auto h) TRLK_INLINE {  // h(values, index of the first)
        blocks_raw([&](const u32x4(&raw)[U], const int(&e)[U]) TRLK_INLINE {
#pragma unroll
            for (int q = 0; q < U; ++q) {
                float v[EPV];
                Elem<DT>::unpack(raw[q], v);
                h(v, uint32_t(e[q]));
            }
        });
    };
    // (where most blocks reach the bound there are thousands of candidates: such a row is passed over as a whole.  1000 rows of 50257 in fp32
    // 44 us instead of 58 with the attempt to list them first)
    const bool too_many = SECOND || (!f.top_k && n_visit > 256 && 2 * n_visit > n_blocks);
    if (!too_many) {
        blocks_raw([&](const u32x4(&raw)[U], const int(&e0)[U]) TRLK_INLINE {
            uint32_t in[U], count = 0;
#pragma unroll
            for (int q = 0; q < U; ++q) {
                float v[EPV];
                Elem<DT>::unpack(raw[q], v);
                in[q] = 0;
#pragma unroll
                for (int e = 0; e < EPV; ++e) in[q] |= in_bound(v[e]) ? 1u << e : 0u;
                count += __popc(in[q]);
            }
            uint32_t to = reserve(&s.n_cand, count);
            // (a lane has one of a vector's logits, two at times: a turn for each, not a branch for each place)
#pragma unroll
            for (int q = 0; q < U; ++q) {
                for (; in[q]; in[q] &= in[q] - 1) {
                    const int e = __builtin_ctz(in[q]);
                    uint32_t key;
                    if constexpr (K::k16) {
                        const uint32_t word = e & 4 ? (e & 2 ? raw[q].w : raw[q].z) : (e & 2 ? raw[q].y : raw[q].x);
                        key = K::of(T(word >> (16 * (e & 1))));
                    } else {
                        key = K::of(__uint_as_float(e & 2 ? (e & 1 ? raw[q].w : raw[q].z) : (e & 1 ? raw[q].y : raw[q].x)));
                    }
                    if (to < kCandidates) s.order[to] = u64(key) << 32 | uint32_t(~(e0[q] + e));
                    ++to;
                }
            }
        });
        __syncthreads();
    }
    const int n_cand = too_many ? kCandidates + 1 : int(s.n_cand);
    // the smallest of the threads' keys, in a word that was ~0
    const auto smallest = [&](uint32_t& word, uint32_t k) TRLK_INLINE {
#pragma unroll
        for (int o = kWave / 2; o > 0; o >>= 1) {
            const uint32_t p = __shfl_xor(k, o);
            k = p < k ? p : k;
        }
        if (lane == 0) atomicMin(&word, k);
        __syncthreads();
        return word;
    };
    uint32_t kept_from = 0;  // the smallest key that min-p keeps
    if (f.min_p > 0.0 && n_cand <= kCandidates) {
        uint32_t k = ~0u;
        for (int i = tid; i < n_cand; i += kSelThreads) {
            const uint32_t q = key_of(s.order[i]);
            if (q < k && key_weight(q) >= f.min_p) k = q;
        }
        kept_from = smallest(s.min_key, k);
    }

    // the integer that a cumulative weight has to pass, and whether it is none (the first kept token passes it then, also one whose
    // weight is less than a unit)
    const auto draw_target = [&](u64 W) TRLK_INLINE {
        const double t = u * double(W);
        const u64 target = t < double(W) ? u64(int64_t(t)) : W - 1;
        return target < W ? target : W - 1;
    };
    // among n <= kPairs kept tokens in s.zone, with their weights, that follow `before`: the one whose cumulative weight in index
    // order passes the target
    const auto draw_from_zone = [&](int n, u64 before, u64 target, u64 W) TRLK_INLINE {
        const Ranked r = rank_pairs(s.zone, s.weight, n, kByIndex);
        const u64 at = before + r.before;
        if (r.real && at <= target && at + r.weight > target) drawn(index_of(r.order), K::to_float(key_of(r.order)), log2_of(W));
    };

    // ---- few candidates: every pair is compared, which gives each one its rank and the mass before it
    if (n_cand <= kPairs) {
        if (tid < n_cand) s.weight[tid] = fixed(key_weight(key_of(s.order[tid])));
        const Ranked r = rank_pairs(s.order, s.weight, n_cand, kByOrder);
        bool kept = r.real && (f.top_k == 0 || r.rank < f.top_k);
        if (f.top_p > 0.0) {
            u64 target = mass_target;
            if (f.top_k) {
                const u64 W1 = block_total(kept ? r.weight : 0, s.slots[1]);
                const double t = __builtin_ceil(f.top_p * double(W1));
                target = t < 1.0 ? u64(1) : u64(int64_t(t));
            }
            kept = kept && r.before < target;
        }
        kept = kept && key_of(r.order) >= kept_from;
        const u64 W = block_total(kept ? r.weight : 0, s.slots[2]);
        if constexpr (SCORE) {
            const int n_kept = __syncthreads_count(kept);  // (a prefix of the order)
            if (r.real && int(r.rank) == n_kept - 1) {
                s.border = key_of(r.order);
                s.border_index = index_of(r.order);
            }
            __syncthreads();
            scored(s.border, s.border_index, [&]() TRLK_INLINE { return log2_of(W); });
        } else {
            const u64 target = draw_target(W);
            if (r.real) {  // (in the order of the ranks, without those that are not kept: their weight is 0)
                s.zone[r.rank] = r.order;
                s.weight[r.rank] = kept ? (target ? r.weight : 1) : 0;
            }
            draw_from_zone(n_cand, 0, target, W);
        }
        return;
    }

    const uint32_t top = K::of_float(m), lowest = K::of_float(-INFINITY) + 1u;
    uint32_t border = 0, border_index = ~0u, at;
    u64 before = 0;
    // ---- some thousands in LDS, one of top-k and top-p (or min-p alone): the border's bin of distances, then the pairs in it; the token's
    // chunk of the row, then the pairs in it
    if (n_cand <= kCandidates && !(f.top_k && f.top_p > 0.0) && bound < kBins) {
        const auto each = [&](auto g) TRLK_INLINE {
            for (int i0 = 0; i0 < n_cand; i0 += kSelThreads) g(i0 + tid < n_cand, i0 + tid < n_cand ? s.order[i0 + tid] : 0);
        };
        const auto bin_of = [&](u64 o) TRLK_INLINE { return distance_bin(m, K::to_float(key_of(o))); };
        bool found = true;
        if (f.top_k || f.top_p > 0.0) {
            clear_bins(s, bound + 1);
            each([&](bool in, u64 o) TRLK_INLINE {
                if (in) atomicAdd(&s.bins[bin_of(o)], f.top_k ? u64(1) : fixed(key_weight(key_of(o))));
            });
            __syncthreads();
            uint32_t bin = 0;
            found = crossing(s, bound + 1, f.top_k ? u64(f.top_k) : mass_target, bin, before);
            if (found) {
                each([&](bool in, u64 o) TRLK_INLINE {
                    in = in && bin_of(o) == int(bin);
                    const uint32_t to = reserve(&s.n_zone, in ? 1 : 0);
                    if (in && to < kPairs) {
                        s.zone[to] = o;
                        s.weight[to] = f.top_k ? u64(1) : fixed(key_weight(key_of(o)));
                    }
                });
                __syncthreads();
                const int n = int(s.n_zone);
                found = n <= kPairs;
                if (found) {
                    const Ranked r = rank_pairs(s.zone, s.weight, n, kByOrder);
                    const bool kept = r.real && before + r.before < (f.top_k ? u64(f.top_k) : mass_target);
                    const int n_kept = __syncthreads_count(kept);
                    if (r.real && int(r.rank) == n_kept - 1) {
                        s.border = key_of(r.order);
                        s.border_index = index_of(r.order);
                    }
                    if (tid == 0) s.n_zone = 0;
                    __syncthreads();
                    border = s.border;
                    border_index = s.border_index;
                }
            }
        }
        if (found) {
            if (kept_from > border) {
                border = kept_from;
                border_index = ~0u;
            }
            const auto kept = [&](u64 o) TRLK_INLINE { return key_of(o) > border || (key_of(o) == border && index_of(o) <= border_index); };
            if constexpr (SCORE) {
                u64 W = 0;
                each([&](bool in, u64 o) TRLK_INLINE {
                    if (in && kept(o)) W += fixed(key_weight(key_of(o)));
                });
                W = block_total(W, s.slots[2]);
                return scored(border, border_index, [&]() TRLK_INLINE { return log2_of(W); });
            } else {
                clear_bins(s, a.chunks);
                each([&](bool in, u64 o) TRLK_INLINE {
                    if (in && kept(o)) atomicAdd(&s.bins[index_of(o) / kChunk], fixed(key_weight(key_of(o))));
                });
                __syncthreads();
                u64 W = 0, target = 0;
                uint32_t bin = 0;
                before = 0;
                crossing_of(s, a.chunks, [&](u64 total) TRLK_INLINE {
                    W = total;
                    target = draw_target(W);
                    return target + 1;
                }, bin, before);
                if (target) {
                    each([&](bool in, u64 o) TRLK_INLINE {
                        in = in && kept(o) && index_of(o) / kChunk == bin;
                        const uint32_t to = reserve(&s.n_zone, in ? 1 : 0);
                        if (in && to < kPairs) {
                            s.zone[to] = o;
                            s.weight[to] = fixed(key_weight(key_of(o)));
                        }
                    });
                    __syncthreads();
                    const int n = int(s.n_zone);
                    if (n <= kPairs) return draw_from_zone(n, before, target, W);
                }
            }
        }
        border = 0;
        border_index = ~0u;
        before = 0;
    }
    // ---- very many candidates, without top-k: two passes over the row.  The first counts the logits in bins linear in them, with their
    // mean in each: that tells the border's bin, or the few where it may be.  The second sums in 64 bits, chunk by chunk,
    // what lies before those bins, and lists what lies in them, where the border is then found.
    if (LONG && n_cand > kCandidates && !f.top_k && x_low > -INFINITY) {
        if (!SECOND && a.longs.count) {  // left to launches of all CUs, if there is a slot
            if (tid == 0) s.bin = atomicAdd(a.longs.count, 1u);
            __syncthreads();
            const uint32_t slot = s.bin;
            if (slot < a.longs.n_slots) {
                LongRow* to = a.longs.at(slot);
                for (int i = tid; i < kBins; i += kSelThreads) to->bins()[i] = 0;
                if (tid == 0) {
                    to->sum = S, to->mass = 0, to->m = m, to->x_low = x_low;
                    to->row = uint32_t(row), to->n_zone = to->done = 0, to->min_key = ~0u;
                }
                return;
            }
        }
        const float scale = bins_per_logit(m, x_low);
        // this workgroup's halves of chunks
        const int half0 = SECOND ? int(blockIdx.x) * kSelWaves : 0, half1 = SECOND && half0 + kSelWaves < 2 * a.chunks ? half0 + kSelWaves : 2 * a.chunks;
        const int64_t v_end = int64_t(half1) * kHalf < V ? int64_t(half1) * kHalf : V;
        // g(values, index of the first) for every vector, end(chunk) after a wave's half of a chunk (waves get as many halves each): 16 logits
        // of a lane at a time, the next in flight
        constexpr int G = 16 / EPV;
        static_assert(kHalf == 16 * kWave && NV == 2 * G, "a half is one set of vectors");
        const auto row_pass = [&](auto g, auto end) TRLK_INLINE {
            const auto load = [&](int64_t e0, u32x4(&q)[G]) TRLK_INLINE {
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const int64_t at = e0 + (i * kWave + lane) * EPV;
                    if (at + EPV <= v_end) {
                        q[i] = *reinterpret_cast<const u32x4_u*>(x + at);
                    } else {
                        float v[EPV];
#pragma unroll
                        for (int e = 0; e < EPV; ++e) v[e] = at + e < v_end ? Elem<DT>::load1(x + at + e) : -INFINITY;
                        q[i] = Elem<DT>::pack(v);
                    }
                }
            };
            u32x4 next[G];
            load(int64_t(half0 + wave) * kHalf, next);
            for (int half = half0 + wave; half < half1; half += kSelWaves) {
                const uint32_t e0 = uint32_t(half) * kHalf;
                u32x4 now[G];
#pragma unroll
                for (int i = 0; i < G; ++i) now[i] = next[i];
                load(int64_t(half + kSelWaves) * kHalf, next);
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    float v[EPV];
                    Elem<DT>::unpack(now[i], v);
                    g(v, e0 + (i * kWave + lane) * EPV);
                    __builtin_amdgcn_sched_barrier(0);
                }
                end(half / 2);
            }
        };
        int zone = kBins, zone_end = kBins;  // [zone, zone_end) has the border
        bool found = true;
        if (f.top_p > 0.0) {
            if constexpr (SECOND) {  // (the launch before this one has counted)
                for (int i = tid; i < kBins; i += kSelThreads) s.bins[i] = left->bins()[i];
            } else {
                clear_bins(s, kBins);
                row_pass([&](const float(&v)[EPV], uint32_t) TRLK_INLINE { count_in_bins(v, m, scale, s.bins); }, [](int) TRLK_INLINE {});
            }
            __syncthreads();
            // how many logits a bin has, times the weight at their mean
            for (int i = tid; i < kBins; i += kSelThreads) {
                const u64 all = s.bins[i];
                const float n = float(uint32_t(all >> 32)), mean = (float(uint32_t(all)) / fmaxf(n, 1.f) + 0.5f) * (1.f / 256.f);
                s.bins[i] = u64(n * fast_exp2(fmaf(-(float(i) + mean) / scale, cf, l2)) + 0.5f);
            }
            __syncthreads();
            // A bin is a hundredth of a power of two wide: a mean stands for its logits to 1e-5 at most, the sums are that good too, and
            // the border lies where they are within 1e-4 of top_p.
            uint32_t bin;
            u64 unused = 0;
            const double p = f.top_p * 0x1p31;
            found = crossing(s, kBins, p > 0x1p31 * 1e-4 ? u64(p - 0x1p31 * 1e-4) + 1 : 1, bin, unused);
            zone = int(bin);
            __syncthreads();
            if (tid == 0) s.bin = ~0u;
            unused = 0;
            zone_end = crossing(s, kBins, u64(p + 0x1p31 * 1e-4) + 1, bin, unused) ? int(bin) + 1 : kBins;
        }
        __syncthreads();
        if (tid == 0) {
            s.n_cand = 0;
            s.min_key = ~0u;
        }
        __syncthreads();
        u64* cmass = reinterpret_cast<u64*>(csum);
        u64 all_mass = 0;
        uint32_t min_key = ~0u;
        if (found) {
            clear_bins(s, a.chunks);  // (of chunks here)
            const float before_zone = float(zone), behind_zone = float(zone_end);
            // (min-p takes away some of what top-p counts)
            const auto second_pass = [&](auto with_min_p) TRLK_INLINE {
                u64 mass = 0;
                row_pass(
                    [&](const float(&v)[EPV], uint32_t e0) TRLK_INLINE {
                        float t[EPV];
                        bool some = false;
#pragma unroll
                        for (int e = 0; e < EPV; ++e) {
                            t[e] = v[e] >= x_low ? (m - v[e]) * scale : INFINITY;
                            some |= t[e] < behind_zone;
                        }
                        if (!__ballot(some)) return;
                        double wd[EPV];
#pragma unroll
                        for (int e = 0; e < EPV; ++e) wd[e] = weight(t[e] < before_zone || with_min_p.value ? v[e] : -INFINITY);
#pragma unroll
                        for (int e = 0; e < EPV; ++e) {
                            u64 w = fixed(wd[e]);
                            if constexpr (with_min_p.value) {
                                w = t[e] < before_zone ? w : 0;
                                all_mass += w;
                                const bool enough = wd[e] >= f.min_p;
                                w = enough ? w : 0;
                                const uint32_t k = K::of_float(v[e]);
                                if (enough && t[e] < behind_zone && k < min_key) min_key = k;
                            }
                            mass += w;
                        }
#pragma unroll
                        for (int e = 0; e < EPV; ++e) {
                            if (t[e] >= before_zone && t[e] < behind_zone) {
                                const uint32_t to = atomicAdd(&s.n_cand, 1u);
                                if (to < kCandidates) s.order[to] = order_of(v[e], e0 + e);
                            }
                        }
                    },
                    [&](int ch) TRLK_INLINE {
                        if constexpr (!with_min_p.value) all_mass += mass;
                        mass = wave_inclusive(mass);
                        if (lane == kWave - 1) atomicAdd(&s.bins[ch], mass);
                        mass = 0;
                    });
            };
            if (f.min_p > 0.0) second_pass(std::true_type{});
            else second_pass(std::false_type{});
            __syncthreads();
            if (SECOND) {
                for (int i = half0 / 2 + tid; i < (half1 + 1) / 2; i += kSelThreads) cmass[i] = s.bins[i];
            } else {
                for (int i = first; i < last; ++i) cmass[i] = s.bins[i];
            }
        }
        min_key = smallest(s.min_key, min_key);
        all_mass = block_total(all_mass, s.slots[1]);
        int n_bin = int(s.n_cand);
        if constexpr (SECOND) {
            if (tid == 0) {
                s.bin = n_bin ? atomicAdd(&left->n_zone, uint32_t(n_bin)) : 0;
                atomicAdd(&left->mass, all_mass);
                atomicMin(&left->min_key, min_key);
            }
            __syncthreads();
            const uint32_t to = s.bin;  // (with more than kCandidates in all, or in one part, nothing of the list is used)
            for (int i = tid; i < n_bin && i < kCandidates; i += kSelThreads)
                if (to + i < kCandidates) left->zone()[to + i] = s.order[i];
            __threadfence();
            __syncthreads();
            if (tid == 0) s.bin = atomicAdd(&left->done, 1u);
            __syncthreads();
            if (s.bin + 1 != uint32_t(a.longs.parts)) return;
            __threadfence();
            all_mass = __hip_atomic_load(&left->mass, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            min_key = __hip_atomic_load(&left->min_key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            n_bin = int(__hip_atomic_load(&left->n_zone, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            for (int i = tid; i < n_bin && i < kCandidates; i += kSelThreads) s.order[i] = left->zone()[i];
            __syncthreads();
        }
        const auto each = [&](auto g) TRLK_INLINE {
            for (int i = tid; i < n_bin; i += kSelThreads) g(key_of(s.order[i]), index_of(s.order[i]));
        };
        bool paired = false;
        if (found && n_bin <= kPairs && f.top_p > 0.0 && all_mass < mass_target) {
            if (tid < n_bin) s.weight[tid] = fixed(key_weight(key_of(s.order[tid])));
            const Ranked r = rank_pairs(s.order, s.weight, n_bin, kByOrder);
            const bool kept = r.real && all_mass + r.before < mass_target;
            const int n_kept = __syncthreads_count(kept);
            if (r.real && int(r.rank) == n_kept - 1) {
                s.border = key_of(r.order);
                s.border_index = index_of(r.order);
                s.before = all_mass + r.before + r.weight;
            }
            __syncthreads();
            paired = n_kept > 0 && s.before >= mass_target;
            if (paired) {
                border = s.border;
                border_index = s.border_index;
            }
            __syncthreads();
        }
        if (found && n_bin <= kCandidates && f.top_p > 0.0 && !paired) {
            before = all_mass;
            found = before < mass_target &&
                    descend(s, [&](auto put) TRLK_INLINE { each([&](uint32_t k, uint32_t) TRLK_INLINE { put(top - k, fixed(key_weight(k))); }); }, 0,
                            top - lowest, mass_target, at, before);
        }
        if (found && n_bin <= kCandidates) {
            kept_from = f.min_p > 0.0 ? min_key : 0u;
            if (f.top_p > 0.0 && !paired) {
                border = top - at;
                const u64 w = fixed(key_weight(border)), ties = (mass_target - before + w - 1) / w;
                u64 count = 0;
                each([&](uint32_t k, uint32_t) TRLK_INLINE { count += k == border; });
                if (ties < block_total(count, s.slots[3])) {
                    before = 0;
                    descend(s, [&](auto put) TRLK_INLINE { each([&](uint32_t k, uint32_t e) TRLK_INLINE { put(e, k == border); }); }, 0, uint32_t(V - 1),
                            ties, border_index, before);
                }
            }
            if (kept_from > border) {
                border = kept_from;
                border_index = ~0u;
            }
            const auto kept = [&](uint32_t k, uint32_t e) TRLK_INLINE { return k > border || (k == border && e <= border_index); };
            // the kept ones of the zone join their chunks
            clear_bins(s, a.chunks);
            each([&](uint32_t k, uint32_t e) TRLK_INLINE {
                if (kept(k, e)) atomicAdd(&s.bins[e / kChunk], fixed(key_weight(k)));
            });
            __syncthreads();
            const auto chunk_mass = [&](int i) TRLK_INLINE { return cmass[i] + s.bins[i]; };
            u64 sum = 0, up, W;
            for (int i = first; i < last; ++i) sum += chunk_mass(i);
            const u64 exc = block_scan(sum, s.slots[2], up, W);
            if constexpr (SCORE) {
                scored(border, border_index, [&]() TRLK_INLINE { return log2_of(W); });
            } else {
                const u64 target = draw_target(W);
                if (exc <= target && up > target) {  // (one thread)
                    u64 run = exc;
                    int ch = first;
                    for (; ch + 1 < last && run + chunk_mass(ch) <= target; ++ch) run += chunk_mass(ch);
                    s.n_list = uint32_t(ch);
                    s.before = run;
                }
                __syncthreads();
                const int64_t e0 = int64_t(s.n_list) * kChunk + tid * PER;
                u64 run = s.before, w[PER], part = 0, all;
                float v[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    v[j] = e0 + j < V ? Elem<DT>::load1(x + e0 + j) : -INFINITY;
                    w[j] = v[j] > -INFINITY && kept(K::of_float(v[j]), uint32_t(e0 + j)) ? fixed(weight(v[j])) : 0;
                    part += w[j];
                }
                run += block_scan(part, s.slots[3], up, all);
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    if (w[j] && run <= target && run + w[j] > target) drawn(e0 + j, v[j], log2_of(W));
                    run += w[j];
                }
            }
            return;
        }
    }

    // ---- the rest: radix descents over the candidates, in LDS or (more of them) read again in each step
    const bool in_lds = n_cand <= kCandidates;
    uint32_t low_key = lowest;
    if (in_lds) {
        uint32_t k = ~0u;
        for (int i = tid; i < n_cand; i += kSelThreads) k = key_of(s.order[i]) < k ? key_of(s.order[i]) : k;
        low_key = smallest(s.low_key, k);
    } else if (f.min_p > 0.0) {
        uint32_t k = ~0u;
        blocks_pass([&](const float(&v)[EPV], uint32_t) TRLK_INLINE {
            for (int e = 0; e < EPV; ++e)
                if (in_bound(v[e]) && weight(v[e]) >= f.min_p && K::of_float(v[e]) < k) k = K::of_float(v[e]);
        });
        kept_from = smallest(s.low_key, k);
    }
    // g(key, index, weight()) for this thread's candidates
    const auto each = [&](auto g) TRLK_INLINE {
        if (in_lds) {
            for (int i = tid; i < n_cand; i += kSelThreads) {
                const u64 o = s.order[i];
                g(key_of(o), index_of(o), [&]() TRLK_INLINE { return fixed(key_weight(key_of(o))); });
            }
        } else {
            blocks_pass([&](const float(&v)[EPV], uint32_t e0) TRLK_INLINE {
#pragma unroll
                for (int e = 0; e < EPV; ++e)
                    if (in_bound(v[e])) g(K::of_float(v[e]), e0 + e, [&]() TRLK_INLINE { return fixed(weight(v[e])); });
            });
        }
    };
    const uint32_t span = top - low_key;
    u64 ties = ~u64(0);  // how many tokens of the border's value are kept
    before = 0;
    if (f.top_k) {
        if (descend(s, [&](auto put) TRLK_INLINE { each([&](uint32_t k, uint32_t, auto) TRLK_INLINE { put(top - k, 1); }); }, 0, span, f.top_k, at, before)) {
            border = top - at;
            ties = f.top_k - before;
        }
    }
    if (f.top_p > 0.0) {
        u64 target = mass_target;
        if (f.top_k) {
            u64 mass = 0;
            each([&](uint32_t k, uint32_t, auto w) TRLK_INLINE {
                if (k > border) mass += w();
            });
            mass = block_total(mass, s.slots[1]);
            if (border) mass += ties * fixed(key_weight(border));
            const double t = __builtin_ceil(f.top_p * double(mass));
            target = t < 1.0 ? u64(1) : u64(int64_t(t));
        }
        before = 0;
        const uint32_t from = border;
        if (descend(s, [&](auto put) TRLK_INLINE {
                each([&](uint32_t k, uint32_t, auto w) TRLK_INLINE {
                    if (k >= from) put(top - k, w());
                });
            }, 0, span, target, at, before)) {
            const uint32_t b = top - at;
            const u64 w = fixed(key_weight(b)), n = (target - before + w - 1) / w;
            ties = b == border && n > ties ? ties : n;
            border = b;
        }
    }
    if (border) {
        u64 count = 0;
        each([&](uint32_t k, uint32_t, auto) TRLK_INLINE { count += k == border; });
        if (ties < block_total(count, s.slots[3])) {
            const uint32_t b = border;
            before = 0;
            descend(s, [&](auto put) TRLK_INLINE { each([&](uint32_t k, uint32_t e, auto) TRLK_INLINE { put(e, k == b); }); }, 0, uint32_t(V - 1), ties,
                    border_index, before);
        }
    }
    if (kept_from > border) {
        border = kept_from;
        border_index = ~0u;
    }
    if (border < lowest) border = lowest;
    const auto kept = [&](uint32_t k, uint32_t e) TRLK_INLINE { return k > border || (k == border && e <= border_index); };
    u64 W = 0;
    each([&](uint32_t k, uint32_t e, auto w) TRLK_INLINE {
        if (kept(k, e)) W += w();
    });
    W = block_total(W, s.slots[2]);
    if constexpr (SCORE) {
        scored(border, border_index, [&]() TRLK_INLINE { return log2_of(W); });
    } else {
        const u64 target = draw_target(W);
        before = 0;
        uint32_t id = 0;
        descend(s, [&](auto put) TRLK_INLINE {
            each([&](uint32_t k, uint32_t e, auto w) TRLK_INLINE {
                if (kept(k, e)) put(e, target ? w() : u64(1));
            });
        }, 0, uint32_t(V - 1), target ? target + 1 : 1, id, before);
        if (tid == 0) drawn(id, Elem<DT>::load1(x + id), log2_of(W));
    }
}

// The first pass over the rows that the selection has left, in parts.
template <int DT>
__global__ __launch_bounds__(kSelThreads) void filter_count_kernel(SelectArgs a) {
    typedef typename Elem<DT>::type T;
    constexpr int EPV = Elem<DT>::EPV, G = 16 / EPV;
    __shared__ u64 bins[kBins];
    if (!a.longs.has(blockIdx.y)) return;
    LongRow* const left = a.longs.at(blockIdx.y);
    const RowFilter f = row_filter(a.f, left->row, a.x.vocab);
    if (!(f.top_p > 0.0)) return;
    const float m = left->m, scale = bins_per_logit(m, left->x_low);
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t e0 = (int64_t(blockIdx.x) * kSelWaves + threadIdx.x / kWave) * kHalf, V = a.x.vocab;
    const T* x = a.x.row<DT>(left->row);
    u32x4 q[G];
    if (e0 < V) load_raw<DT, G>(x + e0, V - e0, lane, q);
    for (int i = threadIdx.x; i < kBins; i += kSelThreads) bins[i] = 0;
    __syncthreads();
    if (e0 < V) {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            float v[EPV];
            Elem<DT>::unpack(q[i], v);
            count_in_bins(v, m, scale, bins);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kSelThreads)
        if (bins[i]) atomicAdd(&left->bins()[i], bins[i]);
}

// ---- backward --------------------------------------------------------------------------------------------------------
struct FilterBwdArgs {
    RowView x;
    int64_t rows;
    int32_t chunks, units_per_row;  // chunks of the forward; waves that a row of the gradient takes
    const int64_t* index;
    double temperature;
    const float* d_temperature;
    const float* state;
    const void* block_max;  // or null: every block is read
    const float* g_logp;
    void* dlogits;  // [rows, vocab]
};

// d logits = g / T * (1[v = token] - kept_v * 2^((x_v - max) * c - log2 W)): the gradient is written once, and only the blocks
// whose maximum reaches the border are read.  Probabilities p = 2^t are in fp32: t is one rounded product and sum, log2 W comes rounded to fp32 from
// the row state, and the power is the hardware's, so p is off by about |t| 2^-23 of itself (9e-7 of a value seen with fp32 logits; far under half a
// step of a 16-bit gradient).  In 64 bits a logit would take 10 operations more of a kernel that the memory bounds.
// A wave's vectors lie at whole cache lines of the gradient, wherever its rows start.  STREAM writes past the caches: for a gradient that they
// cannot hold.  What is left of it in them would be written back under the next scan (4096 rows of 151936 in bf16: scan 181 us after cached
// stores, 130 after these; the gradient itself 202 and 221 us).
template <int DT, bool STREAM>
__global__ __launch_bounds__(kScanThreads) void filter_bwd_kernel(FilterBwdArgs a) {
    typedef typename Elem<DT>::type T;
    constexpr int EPV = Elem<DT>::EPV, NV = kChunk / (kWave * EPV);
    const int lane = threadIdx.x & (kWave - 1);
    const uint32_t unit = __builtin_amdgcn_readfirstlane(int(blockIdx.x * (kScanThreads / kWave) + threadIdx.x / kWave));
    const uint32_t row = unit / uint32_t(a.units_per_row);
    if (row >= a.rows) return;
    const int64_t V = a.x.vocab;
    T* out = static_cast<T*>(a.dlogits) + int64_t(row) * V;
    const int shift = int(reinterpret_cast<uintptr_t>(out) % kLine / sizeof(T));  // entries of the first line that are another row's
    const int64_t first = int64_t(unit - row * uint32_t(a.units_per_row)) * kChunk - shift;
    const float g0 = a.g_logp[row];
    const float bx = a.state[row * int64_t(4)], m = a.state[row * int64_t(4) + 2], l2 = a.state[row * int64_t(4) + 3];
    const uint32_t bi = __float_as_uint(a.state[row * int64_t(4) + 1]);
    double temp = a.d_temperature ? double(a.d_temperature[row]) : a.temperature;
    temp = temp == 0.0 ? 1.0 : temp;
    const float g = float(double(g0) / temp), c = fminf(float(1.4426950408889634074 / temp), FLT_MAX);  // (distances of 0 stay 0)
    const bool too_large = fabsf(g) == INFINITY && fabsf(g0) < INFINITY;  // for fp32, but 0 times it is 0: a temperature of next to nothing
    const bool active = bx < INFINITY && g0 != 0.f;
    const int token = active ? int(a.index[row]) : -1;  // (within the row: the forward has looked)
    const T* x = a.x.row<DT>(row);
    const T* bmax = a.block_max ? static_cast<const T*>(a.block_max) + int64_t(row) * a.chunks * kBlocksPerChunk : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t at = first + (i * kWave + lane) * EPV;
        if (at >= V || at + EPV <= 0) continue;
        const bool whole = at >= 0 && at + EPV <= V;
        float y[EPV];
#pragma unroll
        for (int e = 0; e < EPV; ++e) y[e] = 0.f;
        bool read = active;
        if (active && bmax) {  // (a vector may lie in two blocks)
            const int64_t lo = at < 0 ? 0 : at, hi = at + EPV <= V ? at + EPV - 1 : V - 1;
            read = fmaxf(Elem<DT>::load1(bmax + lo / kBlock), Elem<DT>::load1(bmax + hi / kBlock)) >= bx;
        }
        if (read) {
            float v[EPV];
            if (whole) {
                const u32x4 q = *reinterpret_cast<const u32x4_u*>(x + at);
                Elem<DT>::unpack(q, v);
            } else {
#pragma unroll
                for (int e = 0; e < EPV; ++e) v[e] = at + e >= 0 && at + e < V ? Elem<DT>::load1(x + at + e) : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < EPV; ++e) {
                const int j = int(at) + e;
                const bool kept = v[e] > bx || (v[e] == bx && uint32_t(j) <= bi);
                const float p = kept ? fast_exp2(fmaf(v[e] - m, c, -l2)) : 0.f;
                y[e] = g * ((j == token ? 1.f : 0.f) - p);
            }
            if (too_large) {
#pragma unroll
                for (int e = 0; e < EPV; ++e) y[e] = y[e] == y[e] ? y[e] : 0.f;
            }
        }
        if (whole) {
            u32x4* to = reinterpret_cast<u32x4*>(out + at);
            if constexpr (STREAM)
                __builtin_nontemporal_store(Elem<DT>::pack(y), to);
            else
                *to = Elem<DT>::pack(y);
        } else {
#pragma unroll
            for (int e = 0; e < EPV; ++e)
                if (at + e >= 0 && at + e < V) Elem<DT>::store1(out + at + e, y[e]);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
constexpr double ln2 = 0.69314718055994530942;
double log2e_over(double temperature) { return 1.4426950408889634074 / (temperature == 0.0 ? 1.0 : temperature); }
int64_t chunks_of(int64_t vocab) { return (vocab + kChunk - 1) / kChunk; }
size_t up16(size_t n) { return (n + 15) / 16 * 16; }

int check_filters(const Filters& f, const char* what) {
    TRLK_REQUIRE(f.d_temperature || (f.temperature >= 0.0 && f.temperature <= kMaxTemperature), TRLK_ERR_BAD_VALUE,
                 "%s: temperature must be from 0 to 2^100", what);
    TRLK_REQUIRE(f.d_temperature || f.temperature == 0.0 || 1.4426950408889634074 / f.temperature < INFINITY, TRLK_ERR_BAD_VALUE,
                 "%s: temperature is too small", what);
    TRLK_REQUIRE(f.d_top_p || (f.top_p > 0.0 && f.top_p <= 1.0), TRLK_ERR_BAD_VALUE, "%s: top_p must be in (0, 1]", what);
    TRLK_REQUIRE(f.d_min_p || (f.min_p >= 0.0 && f.min_p <= 1.0), TRLK_ERR_BAD_VALUE, "%s: min_p must be in [0, 1]", what);
    return TRLK_OK;
}

int check_view(const RowView& x, int dtype, int64_t n_seq, const char* what) {
    TRLK_REQUIRE(dtype == TRLK_F32 || dtype == TRLK_BF16 || dtype == TRLK_F16, TRLK_ERR_BAD_DTYPE, "%s: unsupported dtype %d", what, dtype);
    TRLK_REQUIRE(n_seq >= 0 && x.rows_per_seq >= 0 && x.vocab > 0, TRLK_ERR_BAD_SHAPE, "%s: bad shape (%lld sequences, %lld rows, vocab %lld)",
                 what, (long long)n_seq, (long long)x.rows_per_seq, (long long)x.vocab);
    TRLK_REQUIRE(x.vocab <= kMaxVocab, TRLK_ERR_UNSUPPORTED, "%s: vocab %lld is over %lld", what, (long long)x.vocab, (long long)kMaxVocab);
    if (n_seq == 0 || x.rows_per_seq == 0) return TRLK_OK;
    TRLK_REQUIRE(x.rows_per_seq == 1 || x.row_stride >= x.vocab, TRLK_ERR_BAD_STRIDE, "%s: row_stride %lld is less than vocab %lld", what,
                 (long long)x.row_stride, (long long)x.vocab);
    TRLK_REQUIRE(n_seq == 1 || x.seq_stride >= 0, TRLK_ERR_BAD_STRIDE, "%s: negative seq_stride", what);
    // (a launch has fewer than 2^32 threads: 512 for a row, 64 for a chunk of one)
    TRLK_REQUIRE(n_seq < kMaxRows && x.rows_per_seq < kMaxRows && n_seq * x.rows_per_seq < kMaxRows &&
                     n_seq * x.rows_per_seq * (chunks_of(x.vocab) + 1) < kMaxUnits,
                 TRLK_ERR_BAD_SHAPE, "%s: too many rows", what);
    TRLK_REQUIRE(x.logits, TRLK_ERR_NULL_POINTER, "%s: null logits", what);
    TRLK_REQUIRE(reinterpret_cast<uintptr_t>(x.logits) % elem_size(dtype) == 0, TRLK_ERR_BAD_STRIDE, "%s: misaligned logits", what);
    return TRLK_OK;
}

// Which of the scan's outputs the rows' selections may ask for (a value for each row can be anything): block maxima where a filter
// may be in force, sums where a row may have none, or top-p without top-k.
bool needs_blocks(const Filters& f) {
    return f.d_temperature || f.d_top_k || f.d_top_p || f.d_min_p || f.temperature == 0.0 || f.top_k > 0 || f.top_p < 1.0 || f.min_p > 0.0;
}
bool every_top_k(const Filters& f, int64_t vocab) {
    return vocab > 1 && ((!f.d_top_k && f.top_k > 0 && f.top_k < vocab) || (!f.d_temperature && f.temperature == 0.0));
}
// How many rows with more candidates than are held (without top-k, where top-p or min-p bounds them) may be left to the launches of all CUs.
// None where there are more rows than workgroups at a time: so many rows have such ones in every round, and what a round waits for they do
// beside each other.  Mean of 20 draws of logits, with these launches and without: 256 rows of 128257 in bf16 59 and 63 us, 384 of 151936
// in fp32 82 and 95, 1000 of 50257 104 and 71.
int64_t long_rows(int64_t rows, int64_t vocab) { return vocab <= kMaxCandidates || rows > 512 ? 0 : rows < kLongRows ? rows : kLongRows; }
bool may_be_long(const Filters& f, int64_t rows, int64_t vocab) {
    return long_rows(rows, vocab) > 0 && !every_top_k(f, vocab) && (f.d_top_p || f.top_p < 1.0 || f.d_min_p || f.min_p > 0.0);
}
// a top-k whose candidates fit into the variant without LONG only at times (256 rows of 128257 in bf16 with k = 1500: 256 us there, 39 with LONG;
// k = 1000: 26 both)
bool many_top_k(const Filters& f) { return f.top_k > kMaxCandidates / 4 && f.temperature != 0.0; }
bool needs_sums(const Filters& f, int64_t vocab) {
    const bool min_p_alone = !f.d_min_p && f.min_p > 0.0 && !f.d_top_p && f.top_p >= 1.0;
    return !every_top_k(f, vocab) && !min_p_alone;
}

template <int DT>
void launch_scan(const ScanArgs& a, bool sums, bool blocks, hipStream_t stream) {
    const int64_t units = a.rows * a.chunks;
    const dim3 grid(unsigned((units + kScanThreads / kWave - 1) / (kScanThreads / kWave)));
    if (sums && blocks)
        filter_scan_kernel<DT, true, true><<<grid, kScanThreads, 0, stream>>>(a);
    else if (sums)
        filter_scan_kernel<DT, true, false><<<grid, kScanThreads, 0, stream>>>(a);
    else
        filter_scan_kernel<DT, false, true><<<grid, kScanThreads, 0, stream>>>(a);
}

template <int DT>
void launch_select(const SelectArgs& a, bool score, bool any_length, hipStream_t stream) {
    const dim3 grid{unsigned(a.rows)};
    if (score && any_length)
        filter_select_kernel<DT, true, true><<<grid, kSelThreads, 0, stream>>>(a);
    else if (score)
        filter_select_kernel<DT, true, false><<<grid, kSelThreads, 0, stream>>>(a);
    else if (any_length)
        filter_select_kernel<DT, false, true><<<grid, kSelThreads, 0, stream>>>(a);
    else
        filter_select_kernel<DT, false, false><<<grid, kSelThreads, 0, stream>>>(a);
    if (!a.longs.count) return;
    const dim3 parts(unsigned(a.longs.parts), a.longs.n_slots);
    filter_count_kernel<DT><<<parts, kSelThreads, 0, stream>>>(a);
    if (score)
        filter_select_kernel<DT, true, true, true><<<parts, kSelThreads, 0, stream>>>(a);
    else
        filter_select_kernel<DT, false, true, true><<<parts, kSelThreads, 0, stream>>>(a);
}
constexpr size_t kCacheBytes = size_t(256) << 20;  // the last level
template <int DT>
void launch_bwd(const FilterBwdArgs& a, bool past_caches, dim3 grid, hipStream_t stream) {
    if (past_caches)
        filter_bwd_kernel<DT, true><<<grid, kScanThreads, 0, stream>>>(a);
    else
        filter_bwd_kernel<DT, false><<<grid, kScanThreads, 0, stream>>>(a);
}

int run(SelectArgs& a, int dtype, void* workspace, size_t workspace_bytes, void* block_max, bool score, hipStream_t stream, const char* what) {
    const int64_t units = a.rows * a.chunks;
    const bool blocks = needs_blocks(a.f), sums = needs_sums(a.f, a.x.vocab), any_length = !every_top_k(a.f, a.x.vocab) || many_top_k(a.f);
    const size_t sum_bytes = up16(size_t(units) * 8), max_bytes = up16(size_t(units) * 4);
    const size_t need = trlk_token_filter_workspace_bytes(a.rows, a.x.vocab, dtype);
    TRLK_REQUIRE(workspace && workspace_bytes >= need, TRLK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
    TRLK_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, TRLK_ERR_WORKSPACE, "%s: misaligned workspace", what);
    char* ws = static_cast<char*>(workspace);
    a.chunk_sum = reinterpret_cast<double*>(ws);
    a.chunk_max = reinterpret_cast<float*>(ws + sum_bytes);
    if (may_be_long(a.f, a.rows, a.x.vocab)) {
        char* at = ws + sum_bytes + max_bytes + up16(size_t(units) * kBlocksPerChunk * elem_size(dtype));
        at += (64 - reinterpret_cast<uintptr_t>(at) % 64) % 64;
        a.longs = LongRows{reinterpret_cast<uint32_t*>(at), at + 64, uint32_t(long_rows(a.rows, a.x.vocab)), (2 * a.chunks + kSelWaves - 1) / kSelWaves};
    }
    if (!block_max) block_max = ws + sum_bytes + max_bytes;
    a.block_max = block_max;
    a.has_blocks = blocks;
    a.has_sums = sums;
    int bits = 0;
    while ((a.x.vocab >> bits) != 0) ++bits;
    a.fix = 62 - bits < 50 ? 62 - bits : 50;  // a sum of `vocab` weights of at most 1 stays under 2^62
    const ScanArgs sc{a.x, a.rows, a.chunks, a.f, a.row_mask, reinterpret_cast<double*>(ws), reinterpret_cast<float*>(ws + sum_bytes), block_max, a.longs.count};
    switch (dtype) {
        case TRLK_F32:
            launch_scan<TRLK_F32>(sc, sums, blocks, stream);
            launch_select<TRLK_F32>(a, score, any_length, stream);
            break;
        case TRLK_BF16:
            launch_scan<TRLK_BF16>(sc, sums, blocks, stream);
            launch_select<TRLK_BF16>(a, score, any_length, stream);
            break;
        default:
            launch_scan<TRLK_F16>(sc, sums, blocks, stream);
            launch_select<TRLK_F16>(a, score, any_length, stream);
            break;
    }
    return launch_status(what);
}

}  // namespace
}  // namespace trlk

using namespace trlk;

extern "C" int64_t trlk_token_filter_blocks(int64_t vocab) {
    return vocab > 0 && vocab <= kMaxVocab ? chunks_of(vocab) * kBlocksPerChunk : 0;
}
extern "C" int64_t trlk_token_filter_max_vocab(void) { return kMaxVocab; }

extern "C" size_t trlk_token_filter_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
    if (rows <= 0 || vocab <= 0 || vocab > kMaxVocab) return 0;
    const size_t units = size_t(rows) * size_t(chunks_of(vocab));
    const size_t n_long = size_t(long_rows(rows, vocab));
    return up16(units * 8) + up16(units * 4) + up16(units * kBlocksPerChunk * elem_size(dtype)) + (n_long ? 128 + n_long * kLongRowBytes : 0);
}

extern "C" int trlk_sample_tokens(const void* d_logits, int dtype, int64_t n_seq, int64_t rows_per_seq, int64_t vocab,
                                  int64_t seq_stride, int64_t row_stride, const void* d_uniform, int32_t uniform_f64,
                                  double temperature, const float* d_temperature, int64_t top_k, const int32_t* d_top_k, double top_p,
                                  const float* d_top_p, double min_p, const float* d_min_p, const uint8_t* d_row_mask, int64_t fill_id,
                                  int64_t* d_out_ids, float* d_out_logp, int32_t* d_error_flag, void* d_workspace,
                                  size_t workspace_bytes, trlk_stream_t stream) {
    clear_error();
    const Filters f{temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p, d_top_k, log2e_over(temperature), ln2 * (temperature == 0.0 ? 1.0 : temperature)};
    SelectArgs a{};
    a.x = RowView{d_logits, rows_per_seq, vocab, seq_stride, row_stride};
    a.f = f;
    if (const int rc = check_view(a.x, dtype, n_seq, "sample_tokens")) return rc;
    if (const int rc = check_filters(f, "sample_tokens")) return rc;
    a.rows = n_seq * rows_per_seq;
    if (a.rows == 0) return TRLK_OK;
    TRLK_REQUIRE(d_uniform && d_out_ids && d_out_logp, TRLK_ERR_NULL_POINTER, "sample_tokens: null operand");
    a.chunks = int32_t(chunks_of(vocab));
    a.row_mask = d_row_mask;
    a.uniform = d_uniform;
    a.uniform_f64 = uniform_f64;
    a.fill_id = fill_id;
    a.out_ids = d_out_ids;
    a.out_logp = d_out_logp;
    a.error_flag = d_error_flag;
    return run(a, dtype, d_workspace, workspace_bytes, nullptr, false, static_cast<hipStream_t>(stream), "sample_tokens");
}

extern "C" int trlk_filtered_logps_fwd(const void* d_logits, int dtype, int64_t n_seq, int64_t rows_per_seq, int64_t vocab,
                                       int64_t seq_stride, int64_t row_stride, const int64_t* d_index, double temperature,
                                       const float* d_temperature, int64_t top_k, const int32_t* d_top_k, double top_p,
                                       const float* d_top_p, double min_p, const float* d_min_p, const uint8_t* d_row_mask,
                                       float* d_out_logp, float* d_out_state, void* d_out_block_max, int32_t* d_error_flag,
                                       void* d_workspace, size_t workspace_bytes, trlk_stream_t stream) {
    clear_error();
    const Filters f{temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p, d_top_k, log2e_over(temperature), ln2 * (temperature == 0.0 ? 1.0 : temperature)};
    SelectArgs a{};
    a.x = RowView{d_logits, rows_per_seq, vocab, seq_stride, row_stride};
    a.f = f;
    if (const int rc = check_view(a.x, dtype, n_seq, "filtered_logps")) return rc;
    if (const int rc = check_filters(f, "filtered_logps")) return rc;
    a.rows = n_seq * rows_per_seq;
    if (a.rows == 0) return TRLK_OK;
    TRLK_REQUIRE(d_index && d_out_logp && d_out_state, TRLK_ERR_NULL_POINTER, "filtered_logps: null operand");
    // (the selection reads them by vectors: a row has a multiple of 32 of them)
    TRLK_REQUIRE(reinterpret_cast<uintptr_t>(d_out_block_max) % 16 == 0, TRLK_ERR_BAD_STRIDE, "filtered_logps: misaligned block maxima");
    a.chunks = int32_t(chunks_of(vocab));
    a.row_mask = d_row_mask;
    a.index = d_index;
    a.out_state = d_out_state;
    a.out_logp = d_out_logp;
    a.error_flag = d_error_flag;
    return run(a, dtype, d_workspace, workspace_bytes, d_out_block_max, true, static_cast<hipStream_t>(stream), "filtered_logps");
}

extern "C" int trlk_token_filter_has_blocks(double temperature, const float* d_temperature, int64_t top_k, const int32_t* d_top_k,
                                            double top_p, const float* d_top_p, double min_p, const float* d_min_p) {
    return needs_blocks(Filters{temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p, d_top_k, 0.0, 0.0}) ? 1 : 0;
}

extern "C" int trlk_filtered_logps_bwd(const void* d_logits, int dtype, int64_t n_seq, int64_t rows_per_seq, int64_t vocab,
                                       int64_t seq_stride, int64_t row_stride, const int64_t* d_index, double temperature,
                                       const float* d_temperature, const float* d_state, const void* d_block_max, const float* d_g_logp,
                                       void* d_dlogits, trlk_stream_t stream) {
    clear_error();
    FilterBwdArgs a{};
    a.x = RowView{d_logits, rows_per_seq, vocab, seq_stride, row_stride};
    if (const int rc = check_view(a.x, dtype, n_seq, "filtered_logps backward")) return rc;
    TRLK_REQUIRE(d_temperature || (temperature >= 0.0 && temperature <= kMaxTemperature), TRLK_ERR_BAD_VALUE,
                 "filtered_logps backward: temperature must be from 0 to 2^100");
    a.rows = n_seq * rows_per_seq;
    if (a.rows == 0) return TRLK_OK;
    TRLK_REQUIRE(d_index && d_state && d_g_logp && d_dlogits, TRLK_ERR_NULL_POINTER, "filtered_logps backward: null operand");
    TRLK_REQUIRE(reinterpret_cast<uintptr_t>(d_dlogits) % elem_size(dtype) == 0 && reinterpret_cast<uintptr_t>(d_block_max) % elem_size(dtype) == 0,
                 TRLK_ERR_BAD_STRIDE, "filtered_logps backward: misaligned operand");
    a.chunks = int32_t(chunks_of(vocab));
    a.index = d_index;
    a.temperature = temperature;
    a.d_temperature = d_temperature;
    a.state = d_state;
    a.block_max = d_block_max;
    a.g_logp = d_g_logp;
    a.dlogits = d_dlogits;
    const size_t row_bytes = size_t(vocab) * elem_size(dtype);
    const bool lines = row_bytes % kLine == 0 && reinterpret_cast<uintptr_t>(d_dlogits) % kLine == 0;
    a.units_per_row = lines ? a.chunks : int32_t((vocab + kLine / int64_t(elem_size(dtype)) - 1 + kChunk - 1) / kChunk);
    const bool past_caches = row_bytes * size_t(a.rows) > kCacheBytes;
    const dim3 grid(unsigned((a.rows * a.units_per_row + kScanThreads / kWave - 1) / (kScanThreads / kWave)));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == TRLK_F32)
        launch_bwd<TRLK_F32>(a, past_caches, grid, st);
    else if (dtype == TRLK_BF16)
        launch_bwd<TRLK_BF16>(a, past_caches, grid, st);
    else
        launch_bwd<TRLK_F16>(a, past_caches, grid, st);
    return launch_status("filtered_logps backward");
}
