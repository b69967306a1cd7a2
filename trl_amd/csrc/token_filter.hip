// K8: tokens drawn from, and scored under, softmax(logits / T) after top-k, top-p and min-p.
//
// Order of a row's tokens: logit descending, index ascending.  All three filters keep a prefix of that order (top-k the first k,
// top-p those before which less than top_p of the mass lies that top-k kept, min-p those of weight >= min_p, the largest being 1),
// so what a row keeps is one border: a value, and among the tokens of exactly that value the last index.  With
// w_v = exp((x_v - max) / T) for the kept tokens, a token is drawn as the first index whose cumulative weight exceeds u * W.
//
// Two launches.  filter_scan_kernel reads the logits once, a wave per chunk of 2048, and leaves the chunk's maximum, its sum of
// weights in 64 bits and the maximum of every block of 64 logits.  filter_select_kernel has one workgroup per row: the block
// maxima bound the border from below (the k-th largest of them is at most the k-th largest logit; blocks whose maxima hold
// top_p of the mass hold the tokens of top-p), so that only blocks with a maximum over that bound are read again -- a few dozen of
// some thousand -- and the border, the kept mass and the token come from those candidates.
//
// Whole numbers come out, and the same ones whatever the launch: sums of weights are 64-bit floats in a fixed order over a row's
// chunks, or 64-bit integers (weights in units of 2^-fix, whose sums do not depend on the order in which threads add them).
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
constexpr int kCandidates = 2048;            // that are kept in LDS; rows with more read their blocks again in every step
constexpr int kList = 2048;                  // blocks over the bound that are listed; with more every block is looked at
constexpr int64_t kMaxVocab = int64_t(1) << 22;

typedef unsigned long long u64;
typedef u32x4 u32x4_u __attribute__((aligned(2)));  // a 16-byte vector at any element alignment

// ---- weights ---------------------------------------------------------------------------------------------------------
// 2^t for t <= 0 in 64 bits: 2^(t - n) on [-1/2, 1/2] by a polynomial of degree 9 that interpolates it at the Chebyshev points
// (relative error 3e-14), times 2^n.  -inf and everything under -1100 give 0.
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

// maximum that lets a NaN through
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float wave_max_nan(float v) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor(v, o));
    return v;
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
};
struct RowFilter {
    double c;         // log2(e) / T
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
    r.ok = T >= 0.0 && T < INFINITY && p == p && q == q;
    if (T == 0.0) {
        T = 1.0;
        k = 1;
    }
    r.c = 1.4426950408889634074 / T;
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
    __device__ __forceinline__ const typename Elem<DT>::type* row(int64_t r) const {
        const int64_t b = r / rows_per_seq, t = r - b * rows_per_seq;
        return static_cast<const typename Elem<DT>::type*>(logits) + b * seq_stride + t * row_stride;
    }
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
};

// The VEC = kChunk / (64 * EPV) vectors of a lane: vector i holds the logits (i * 64 + lane) * EPV on of the chunk.  What lies behind
// the row's end is -inf.
template <int DT, int NV>
__device__ __forceinline__ void load_chunk(const typename Elem<DT>::type* p, int n, int lane, float (&x)[NV * Elem<DT>::EPV]) {
    constexpr int EPV = Elem<DT>::EPV;
    if (n == kChunk) {
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

template <int DT, bool SUMS, bool BLOCKS>
__global__ __launch_bounds__(kScanThreads) void filter_scan_kernel(ScanArgs a) {
    typedef typename Elem<DT>::type T;
    constexpr int EPV = Elem<DT>::EPV, NV = kChunk / (kWave * EPV), LPB = kBlock / EPV;  // LPB: lanes of a block
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t unit = __builtin_amdgcn_readfirstlane(int(blockIdx.x * (kScanThreads / kWave) + threadIdx.x / kWave));
    const int64_t row = unit / a.chunks;
    if (row >= a.rows) return;
    const int chunk = int(unit - row * a.chunks);
    if (a.row_mask && a.row_mask[row] == 0) return;
    const T* p = a.x.row<DT>(row) + int64_t(chunk) * kChunk;
    const int64_t left = a.x.vocab - int64_t(chunk) * kChunk;
    float x[NV * EPV];
    load_chunk<DT, NV>(p, left < kChunk ? int(left) : kChunk, lane, x);
    float m = -INFINITY, mine = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float v = x[i * EPV];
#pragma unroll
        for (int e = 1; e < EPV; ++e) v = max_nan(v, x[i * EPV + e]);
        if constexpr (BLOCKS) {
#pragma unroll
            for (int o = 1; o < LPB; o <<= 1) v = max_nan(v, __shfl_xor(v, o));
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
        const double c = row_filter(a.f, row, a.x.vocab).c, ref = m > -INFINITY && m < INFINITY ? double(m) : 0.0;
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < NV * EPV; ++j) s += exp2_f64((double(x[j]) - ref) * c);
#pragma unroll
        for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) a.chunk_sum[unit] = s;
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
    const double* chunk_sum;
    const float* chunk_max;
    const void* block_max;
    const void* uniform;  // sample: fp32 or fp64 [rows]
    int32_t uniform_f64;
    int64_t fill_id;
    int64_t* out_ids;
    const int64_t* index;  // score: [rows]
    float* out_state;      // score: [rows, 4]: border value, border index (bits), maximum, log2 of the kept mass in units of its weight
    float* out_logp;
    int32_t* error_flag;
};

struct SelectShared {
    u64 bins[kBins];
    u64 weight[kCandidates];
    uint32_t key[kCandidates], index[kCandidates];
    uint16_t list[kList];
    u64 scan[kSelWaves];
    double scan_f[kSelWaves];
    float wave_f[kSelWaves];
    u64 before;
    double prefix;
    uint32_t bin, n_list, n_cand, min_key, lo, hi;
};

template <typename V>
__device__ __forceinline__ V wave_inclusive(V v, int lane) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const V u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}
// Sum over the threads before this one; `total` over all.  Contains two barriers.
template <typename V>
__device__ __forceinline__ V block_exclusive(V v, V* scratch, V& total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const V inc = wave_inclusive(v, lane);
    __syncthreads();
    if (lane == kWave - 1) scratch[wave] = inc;
    __syncthreads();
    V base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
        if (w == wave) base = all;
        all += scratch[w];
    }
    total = all;
    return base + (inc - v);
}
__device__ __forceinline__ u64 block_total(u64 v, u64* scratch) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    u64 r = 0;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) r += scratch[w];
    return r;
}

// The smallest position in [lo, hi] up to which `before` and the values reach `target`, and in `before` what lies before it.
// `each(f)` calls f(position, value) for this thread's share of the items.  False if all of them do not reach it.
template <typename Each>
__device__ bool descend(SelectShared& s, Each each, uint32_t lo, uint32_t hi, u64 target, uint32_t& position, u64& before) {
    for (;;) {
        const uint32_t span = hi - lo;
        const int bits = span ? 32 - __builtin_clz(span) : 0, shift = bits > kBinBits ? bits - kBinBits : 0;
        const int n = int(span >> shift) + 1;
        for (int i = threadIdx.x; i < n; i += kSelThreads) s.bins[i] = 0;
        __syncthreads();
        if (threadIdx.x == 0) s.bin = ~0u;  // (everyone has read the last step's; the next is written two barriers from here)
        each([&](uint32_t at, u64 value) {
            if (at >= lo && at <= hi && value) atomicAdd(&s.bins[(at - lo) >> shift], value);
        });
        __syncthreads();
        u64 v[4], sum = 0, total;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = 4 * threadIdx.x + j;
            v[j] = i < n ? s.bins[i] : 0;
            sum += v[j];
        }
        u64 at = before + block_exclusive(sum, s.scan, total);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (at < target && at + v[j] >= target) {  // (one bin of one thread)
                s.bin = 4 * threadIdx.x + j;
                s.before = at;
            }
            at += v[j];
        }
        __syncthreads();
        const uint32_t bin = s.bin;
        if (bin == ~0u) return false;
        before = s.before;
        lo += bin << shift;
        position = lo;
        if (shift == 0) return true;
        const uint32_t last = lo + ((1u << shift) - 1u);
        hi = last < hi ? last : hi;
    }
}

template <int DT, bool SCORE>
__global__ __launch_bounds__(kSelThreads) void filter_select_kernel(SelectArgs a) {
    typedef typename Elem<DT>::type T;
    typedef Key<DT> K;
    __shared__ SelectShared s;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int64_t row = blockIdx.x, V = a.x.vocab;
    if (a.row_mask && a.row_mask[row] == 0) {
        if (tid == 0) {
            if constexpr (SCORE) {
                a.out_state[row * 4] = INFINITY;
                a.out_state[row * 4 + 1] = a.out_state[row * 4 + 2] = a.out_state[row * 4 + 3] = 0.f;
            } else {
                a.out_ids[row] = a.fill_id;
            }
            a.out_logp[row] = 0.f;
        }
        return;
    }
    const RowFilter f = row_filter(a.f, row, V);
    const T* x = a.x.row<DT>(row);
    const float* cmax = a.chunk_max + row * a.chunks;
    const double* csum = a.chunk_sum + row * a.chunks;

    // the row's maximum
    float m = -INFINITY;
    for (int i = tid; i < a.chunks; i += kSelThreads) m = max_nan(m, cmax[i]);
    m = wave_max_nan(m);
    if (lane == 0) s.wave_f[wave] = m;
    if (tid == 0) {
        s.n_list = s.n_cand = 0;
        s.min_key = ~0u;
        s.lo = ~0u;
        s.hi = 0;
    }
    __syncthreads();
    m = s.wave_f[0];
#pragma unroll
    for (int w = 1; w < kSelWaves; ++w) m = max_nan(m, s.wave_f[w]);
    int64_t token = 0;
    bool token_ok = true;
    if constexpr (SCORE) {
        token = a.index[row];
        token_ok = token >= 0 && token < V;
        if (!token_ok && tid == 0 && a.error_flag) atomicOr(a.error_flag, TRLK_FLAG_INDEX_OUT_OF_RANGE);
    }
    if (!f.ok || !(m < INFINITY) || m == -INFINITY) {  // no distribution
        if (tid == 0) {
            if constexpr (SCORE) {
                a.out_state[row * 4] = INFINITY;
                a.out_state[row * 4 + 1] = a.out_state[row * 4 + 2] = a.out_state[row * 4 + 3] = 0.f;
            } else {
                a.out_ids[row] = -1;
            }
            a.out_logp[row] = NAN;
            if (a.error_flag) atomicOr(a.error_flag, TRLK_FLAG_NO_DISTRIBUTION);
        }
        return;
    }
    double u = 0.0;
    if constexpr (!SCORE) {
        u = a.uniform_f64 ? static_cast<const double*>(a.uniform)[row] : double(static_cast<const float*>(a.uniform)[row]);
        u = u > 0.0 ? u : 0.0;  // (and NaN)
    }
    const double c = f.c, ref = double(m), unit = __builtin_amdgcn_ldexp(1.0, a.fix);
    const auto weight = [&](float v) { return exp2_f64((double(v) - ref) * c); };
    const auto fixed = [&](double w) { return u64(int64_t(__builtin_rint(w * unit))); };

    // the row's sum of weights, and this thread's chunks' place in it
    const bool filtered = f.top_k || f.top_p > 0.0 || f.min_p > 0.0;
    double S = 0.0, mine = 0.0, base = 0.0;
    const int per = (a.chunks + kSelThreads - 1) / kSelThreads, first = tid * per,
              last = first + per < a.chunks ? first + per : a.chunks;
    if (!filtered || (f.top_p > 0.0 && !f.top_k)) {
        for (int i = first; i < last; ++i) mine += csum[i] * weight(cmax[i]);
        base = block_exclusive(mine, s.scan_f, S);
    }

    uint32_t border = 0, border_index = ~0u;  // everything
    double log2_mass;
    int64_t id = 0;
    if (!filtered) {
        log2_mass = log2(S);
        if constexpr (!SCORE) {
            const double target = u * S;
            double at = base;
            for (int i = first; i < last; ++i) {
                const double v = csum[i] * weight(cmax[i]);
                if (v > 0.0) atomicMax(&s.hi, uint32_t(i));
                if (at + v > target) {
                    atomicMin(&s.lo, uint32_t(i));
                    break;
                }
                at += v;
            }
            __syncthreads();
            const int chunk = s.lo != ~0u ? int(s.lo) : int(s.hi);  // (u * S rounded up to the whole sum: the last one)
            if (chunk >= first && chunk < last) {
                double before = base;
                for (int i = first; i < chunk; ++i) before += csum[i] * weight(cmax[i]);
                s.prefix = before;
            }
            __syncthreads();
            const double prefix = s.prefix;
            if (tid == 0) {
                s.lo = ~0u;
                s.hi = 0;
            }
            constexpr int PER = kChunk / kSelThreads;
            double w[PER], sum = 0.0, all;
            const int64_t e0 = int64_t(chunk) * kChunk + tid * PER;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                w[j] = e0 + j < V ? weight(Elem<DT>::load1(x + e0 + j)) : 0.0;
                sum += w[j];
            }
            double run = prefix + block_exclusive(sum, s.scan_f, all);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                run += w[j];
                if (w[j] > 0.0) {
                    atomicMax(&s.hi, uint32_t(e0 + j));
                    if (run > target) atomicMin(&s.lo, uint32_t(e0 + j));
                }
            }
            __syncthreads();
            id = s.lo != ~0u ? s.lo : s.hi;
        }
    } else {
        const T* bmax = static_cast<const T*>(a.block_max) + row * a.chunks * kBlocksPerChunk;
        const int n_blocks = int((V + kBlock - 1) / kBlock);
        const uint32_t top = K::of_float(m), lowest = K::of_float(-INFINITY) + 1u;
        // a bound under the border, as a key and as a value
        uint32_t bound = lowest, at;
        float x_bound = -INFINITY;
        u64 before = 0;
        const u64 mass_target = [&] {  // of top-p without top-k
            const double t = __builtin_ceil(f.top_p * S * unit);
            return t < 1.0 ? u64(1) : u64(int64_t(t));
        }();
        if (f.top_k) {
            if (f.top_k <= uint32_t(n_blocks) &&
                descend(s, [&](auto put) {
                    for (int i = tid; i < n_blocks; i += kSelThreads) {
                        const uint32_t k = K::of(bmax[i]);
                        if (k >= lowest) put(top - k, 1);
                    }
                }, 0, top - lowest, f.top_k, at, before))
                bound = top - at;
        } else if (f.top_p > 0.0) {
            // (the sum of rounded weights may be half a unit for each block too large)
            if (descend(s, [&](auto put) {
                    for (int i = tid; i < n_blocks; i += kSelThreads) {
                        const uint32_t k = K::of(bmax[i]);
                        if (k >= lowest) put(top - k, fixed(weight(K::to_float(k))));
                    }
                }, 0, top - lowest, mass_target + n_blocks, at, before)) {
                bound = top - at;
            } else {  // all tokens of less than (1 - top_p) / V of the mass together have less than 1 - top_p
                const double e = (1.0 - f.top_p) * S / double(V) * (1.0 - 1e-9);
                x_bound = float(ref + log2(e) / c);
                x_bound -= 1e-6f * fabsf(x_bound) + 1e-30f;
            }
        }
        if (f.min_p > 0.0 && !(f.top_k && f.top_p > 0.0)) {  // (top-p of top-k counts what min-p takes away)
            float b = float(ref + log2(f.min_p) / c);
            b -= 1e-6f * fabsf(b) + 1e-30f;
            x_bound = fmaxf(x_bound, b);
        }
        // blocks over the bound
        const auto block_in = [&](int i) {
            const uint32_t k = K::of(bmax[i]);
            return k >= bound && K::to_float(k) >= x_bound;
        };
        __syncthreads();
        for (int i = tid; i < n_blocks; i += kSelThreads) {
            if (block_in(i)) {
                const uint32_t to = atomicAdd(&s.n_list, 1u);
                if (to < kList) s.list[to] = uint16_t(i);
            }
        }
        __syncthreads();
        const bool listed = s.n_list <= kList;
        const int n_visit = listed ? int(s.n_list) : n_blocks;
        // all logits over the bound, a wave to a block: g(valid, key, index), with all lanes of the wave in it
        const auto stream = [&](auto g) {
            for (int j = wave; j < n_visit; j += kSelWaves) {
                const int blk = listed ? int(s.list[j]) : j;
                if (!listed && !block_in(blk)) continue;
                const int64_t e = int64_t(blk) * kBlock + lane;
                const uint32_t k = e < V ? K::of(x[e]) : 0u;
                g(e < V && k >= bound && K::to_float(k) >= x_bound, k, uint32_t(e));
            }
        };
        uint32_t min_key = ~0u;
        stream([&](bool in, uint32_t k, uint32_t e) {
            const u64 vote = __ballot(in);
            uint32_t to = 0;
            if (lane == 0 && vote) to = atomicAdd(&s.n_cand, uint32_t(__popcll(vote)));
            to = __shfl(to, 0) + __popcll(vote & ((u64(1) << lane) - 1));
            if (in) {
                const double w = weight(K::to_float(k));
                if (w >= f.min_p && k < min_key) min_key = k;
                if (to < kCandidates) {
                    s.key[to] = k;
                    s.index[to] = e;
                    s.weight[to] = fixed(w);
                }
            }
        });
        if (f.min_p > 0.0 && min_key != ~0u) atomicMin(&s.min_key, min_key);
        __syncthreads();
        const int n_cand = int(s.n_cand);
        const uint32_t kept_from = f.min_p > 0.0 ? s.min_key : 0u;
        const bool in_lds = n_cand <= kCandidates;
        // g(key, index, weight) for this thread's candidates
        const auto each = [&](auto g) {
            if (in_lds) {
                for (int i = tid; i < n_cand; i += kSelThreads) g(s.key[i], s.index[i], [&] { return s.weight[i]; });
            } else {
                stream([&](bool in, uint32_t k, uint32_t e) {
                    if (in) g(k, e, [&] { return fixed(weight(K::to_float(k))); });
                });
            }
        };
        const uint32_t span = top - lowest;
        u64 ties = ~u64(0);  // how many tokens of the border's value are kept
        if (f.top_k) {
            before = 0;
            if (descend(s, [&](auto put) { each([&](uint32_t k, uint32_t, auto) { put(top - k, 1); }); }, 0, span, f.top_k, at, before)) {
                border = top - at;
                ties = f.top_k - before;
            }
        }
        if (f.top_p > 0.0) {
            u64 target = mass_target;
            if (f.top_k) {
                u64 mass = 0;
                each([&](uint32_t k, uint32_t, auto w) {
                    if (k > border) mass += w();
                });
                mass = block_total(mass, s.scan);
                if (border) mass += ties * fixed(weight(K::to_float(border)));
                const double t = __builtin_ceil(f.top_p * double(mass));
                target = t < 1.0 ? u64(1) : u64(int64_t(t));
            }
            before = 0;
            const uint32_t from = border;
            if (descend(s, [&](auto put) {
                    each([&](uint32_t k, uint32_t, auto w) {
                        if (k >= from) put(top - k, w());
                    });
                }, 0, span, target, at, before)) {
                const uint32_t b = top - at;
                const u64 w = fixed(weight(K::to_float(b))), n = (target - before + w - 1) / w;
                ties = b == border && n > ties ? ties : n;
                border = b;
            }
        }
        if (border) {
            u64 count = 0;
            each([&](uint32_t k, uint32_t, auto) { count += k == border; });
            if (ties < block_total(count, s.scan)) {
                const uint32_t b = border;
                before = 0;
                descend(s, [&](auto put) { each([&](uint32_t k, uint32_t e, auto) { put(e, k == b); }); }, 0, uint32_t(V - 1), ties,
                        border_index, before);
            }
        }
        if (kept_from > border) {
            border = kept_from;
            border_index = ~0u;
        }
        if (border < lowest) border = lowest;
        const auto kept = [&](uint32_t k, uint32_t e) { return k > border || (k == border && e <= border_index); };
        u64 W = 0;
        each([&](uint32_t k, uint32_t e, auto w) {
            if (kept(k, e)) W += w();
        });
        W = block_total(W, s.scan);
        log2_mass = log2(double(W)) - a.fix;
        if constexpr (!SCORE) {
            double t = u * double(W);
            u64 target = t < double(W) ? u64(int64_t(t)) : W - 1;
            target = target < W ? target : W - 1;
            before = 0;
            uint32_t e_at = 0;
            // (a target of 0 is reached by the first kept token, also by one whose weight is less than a unit)
            descend(s, [&](auto put) {
                each([&](uint32_t k, uint32_t e, auto w) {
                    if (kept(k, e)) put(e, target ? w() : u64(1));
                });
            }, 0, uint32_t(V - 1), target ? target + 1 : 1, e_at, before);
            id = e_at;
        }
    }

    if (tid != 0) return;
    if constexpr (SCORE) {
        const float bx = filtered ? K::to_float(border) : -INFINITY;
        float logp = NAN;
        bool inside = false;
        if (token_ok) {
            const T raw = x[token];
            const float v = Elem<DT>::to_float(raw);
            const uint32_t k = K::of(raw);
            inside = v > -INFINITY && (!filtered || k > border || (k == border && uint32_t(token) <= border_index));
            logp = inside ? float(((double(v) - ref) * c - log2_mass) * 0.69314718055994530942) : -INFINITY;
        }
        float* st = a.out_state + row * 4;
        st[0] = inside ? bx : INFINITY;  // (no gradient reaches a row whose token lies outside)
        st[1] = __uint_as_float(border_index);
        st[2] = m;
        st[3] = float(log2_mass);
        a.out_logp[row] = logp;
    } else {
        a.out_ids[row] = id;
        const float v = Elem<DT>::load1(x + id);
        a.out_logp[row] = float(((double(v) - ref) * c - log2_mass) * 0.69314718055994530942);
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------
struct FilterBwdArgs {
    RowView x;
    int64_t rows;
    int32_t chunks;
    const int64_t* index;
    double temperature;
    const float* d_temperature;
    const float* state;
    const void* block_max;  // or null: every block is read
    const float* g_logp;
    void* dlogits;  // [rows, vocab]
};

// d logits = g / T * (1[v = token] - kept_v * 2^((x_v - max) * c - log2 W)): the gradient is written once, and only the blocks
// whose maximum reaches the border are read.
template <int DT>
__global__ __launch_bounds__(kScanThreads) void filter_bwd_kernel(FilterBwdArgs a) {
    typedef typename Elem<DT>::type T;
    constexpr int EPV = Elem<DT>::EPV, NV = kChunk / (kWave * EPV), LPB = kBlock / EPV;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t unit = __builtin_amdgcn_readfirstlane(int(blockIdx.x * (kScanThreads / kWave) + threadIdx.x / kWave));
    const int64_t row = unit / a.chunks;
    if (row >= a.rows) return;
    const int chunk = int(unit - row * a.chunks);
    const int64_t V = a.x.vocab, e0 = int64_t(chunk) * kChunk;
    const int n = V - e0 < kChunk ? int(V - e0) : kChunk;
    const float g0 = a.g_logp[row];
    const float bx = a.state[row * 4], m = a.state[row * 4 + 2], l2 = a.state[row * 4 + 3];
    const uint32_t bi = __float_as_uint(a.state[row * 4 + 1]);
    double temp = a.d_temperature ? double(a.d_temperature[row]) : a.temperature;
    temp = temp == 0.0 ? 1.0 : temp;
    const float g = float(double(g0) / temp), c = float(1.4426950408889634074 / temp);
    const bool active = bx < INFINITY && g0 != 0.f;
    const int token = active ? int(a.index[row] - e0) : -1;  // (within the row: the forward has looked)
    const T* x = a.x.row<DT>(row) + e0;
    T* out = static_cast<T*>(a.dlogits) + row * V + e0;
    const T* bmax = a.block_max ? static_cast<const T*>(a.block_max) + unit * kBlocksPerChunk : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * kWave + lane) * EPV;
        float y[EPV];
#pragma unroll
        for (int e = 0; e < EPV; ++e) y[e] = 0.f;
        if (active && at < n && (!bmax || Elem<DT>::load1(bmax + i * (kWave / LPB) + lane / LPB) >= bx)) {
            float v[EPV];
            if (at + EPV <= n) {
                const u32x4 q = *reinterpret_cast<const u32x4_u*>(x + at);
                Elem<DT>::unpack(q, v);
            } else {
#pragma unroll
                for (int e = 0; e < EPV; ++e) v[e] = at + e < n ? Elem<DT>::load1(x + at + e) : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < EPV; ++e) {
                const bool kept = v[e] > bx || (v[e] == bx && uint32_t(e0 + at + e) <= bi);
                const float p = kept ? fast_exp2(fmaf(v[e] - m, c, -l2)) : 0.f;
                y[e] = g * ((at + e == token ? 1.f : 0.f) - p);
            }
        }
        if (at + EPV <= n) {
            *reinterpret_cast<u32x4_u*>(out + at) = Elem<DT>::pack(y);
        } else {
#pragma unroll
            for (int e = 0; e < EPV; ++e)
                if (at + e < n) Elem<DT>::store1(out + at + e, y[e]);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
int64_t chunks_of(int64_t vocab) { return (vocab + kChunk - 1) / kChunk; }
size_t up16(size_t n) { return (n + 15) / 16 * 16; }

int check_filters(const Filters& f, const char* what) {
    TRLK_REQUIRE(f.d_temperature || (f.temperature >= 0.0 && f.temperature < INFINITY), TRLK_ERR_BAD_VALUE,
                 "%s: temperature must be >= 0 and finite", what);
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
    TRLK_REQUIRE(n_seq < (int64_t(1) << 31) && x.rows_per_seq < (int64_t(1) << 31) &&
                     n_seq * x.rows_per_seq < (int64_t(1) << 31) / chunks_of(x.vocab) - 8,
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
bool needs_sums(const Filters& f, int64_t vocab) {
    const bool every_k = vocab > 1 && ((!f.d_top_k && f.top_k > 0 && f.top_k < vocab) || (!f.d_temperature && f.temperature == 0.0));
    const bool min_p_alone = !f.d_min_p && f.min_p > 0.0 && !f.d_top_p && f.top_p >= 1.0;
    return !every_k && !min_p_alone;
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

int run(SelectArgs& a, int dtype, void* workspace, size_t workspace_bytes, void* block_max, bool score, hipStream_t stream, const char* what) {
    const int64_t units = a.rows * a.chunks;
    const bool blocks = needs_blocks(a.f), sums = needs_sums(a.f, a.x.vocab);
    const size_t sum_bytes = up16(size_t(units) * 8), max_bytes = up16(size_t(units) * 4);
    const size_t need = trlk_token_filter_workspace_bytes(a.rows, a.x.vocab, dtype);
    TRLK_REQUIRE(workspace && workspace_bytes >= need, TRLK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
    TRLK_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, TRLK_ERR_WORKSPACE, "%s: misaligned workspace", what);
    char* ws = static_cast<char*>(workspace);
    a.chunk_sum = reinterpret_cast<double*>(ws);
    a.chunk_max = reinterpret_cast<float*>(ws + sum_bytes);
    if (!block_max) block_max = ws + sum_bytes + max_bytes;
    a.block_max = block_max;
    int bits = 0;
    while ((a.x.vocab >> bits) != 0) ++bits;
    a.fix = 62 - bits;  // a sum of `vocab` weights of at most 1 stays under 2^62
    const ScanArgs sc{a.x, a.rows, a.chunks, a.f, a.row_mask, reinterpret_cast<double*>(ws), reinterpret_cast<float*>(ws + sum_bytes), block_max};
    const dim3 grid{unsigned(a.rows)};
    switch (dtype) {
        case TRLK_F32:
            launch_scan<TRLK_F32>(sc, sums, blocks, stream);
            score ? filter_select_kernel<TRLK_F32, true><<<grid, kSelThreads, 0, stream>>>(a)
                  : filter_select_kernel<TRLK_F32, false><<<grid, kSelThreads, 0, stream>>>(a);
            break;
        case TRLK_BF16:
            launch_scan<TRLK_BF16>(sc, sums, blocks, stream);
            score ? filter_select_kernel<TRLK_BF16, true><<<grid, kSelThreads, 0, stream>>>(a)
                  : filter_select_kernel<TRLK_BF16, false><<<grid, kSelThreads, 0, stream>>>(a);
            break;
        default:
            launch_scan<TRLK_F16>(sc, sums, blocks, stream);
            score ? filter_select_kernel<TRLK_F16, true><<<grid, kSelThreads, 0, stream>>>(a)
                  : filter_select_kernel<TRLK_F16, false><<<grid, kSelThreads, 0, stream>>>(a);
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
    return up16(units * 8) + up16(units * 4) + up16(units * kBlocksPerChunk * elem_size(dtype));
}

extern "C" int trlk_sample_tokens(const void* d_logits, int dtype, int64_t n_seq, int64_t rows_per_seq, int64_t vocab,
                                  int64_t seq_stride, int64_t row_stride, const void* d_uniform, int32_t uniform_f64,
                                  double temperature, const float* d_temperature, int64_t top_k, const int32_t* d_top_k, double top_p,
                                  const float* d_top_p, double min_p, const float* d_min_p, const uint8_t* d_row_mask, int64_t fill_id,
                                  int64_t* d_out_ids, float* d_out_logp, int32_t* d_error_flag, void* d_workspace,
                                  size_t workspace_bytes, trlk_stream_t stream) {
    clear_error();
    const Filters f{temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p, d_top_k};
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
    const Filters f{temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p, d_top_k};
    SelectArgs a{};
    a.x = RowView{d_logits, rows_per_seq, vocab, seq_stride, row_stride};
    a.f = f;
    if (const int rc = check_view(a.x, dtype, n_seq, "filtered_logps")) return rc;
    if (const int rc = check_filters(f, "filtered_logps")) return rc;
    a.rows = n_seq * rows_per_seq;
    if (a.rows == 0) return TRLK_OK;
    TRLK_REQUIRE(d_index && d_out_logp && d_out_state, TRLK_ERR_NULL_POINTER, "filtered_logps: null operand");
    TRLK_REQUIRE(reinterpret_cast<uintptr_t>(d_out_block_max) % elem_size(dtype) == 0, TRLK_ERR_BAD_STRIDE, "filtered_logps: misaligned block maxima");
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
    return needs_blocks(Filters{temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p, d_top_k}) ? 1 : 0;
}

extern "C" int trlk_filtered_logps_bwd(const void* d_logits, int dtype, int64_t n_seq, int64_t rows_per_seq, int64_t vocab,
                                       int64_t seq_stride, int64_t row_stride, const int64_t* d_index, double temperature,
                                       const float* d_temperature, const float* d_state, const void* d_block_max, const float* d_g_logp,
                                       void* d_dlogits, trlk_stream_t stream) {
    clear_error();
    FilterBwdArgs a{};
    a.x = RowView{d_logits, rows_per_seq, vocab, seq_stride, row_stride};
    if (const int rc = check_view(a.x, dtype, n_seq, "filtered_logps backward")) return rc;
    TRLK_REQUIRE(d_temperature || (temperature >= 0.0 && temperature < INFINITY), TRLK_ERR_BAD_VALUE,
                 "filtered_logps backward: temperature must be >= 0 and finite");
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
    const dim3 grid(unsigned((a.rows * a.chunks + kScanThreads / kWave - 1) / (kScanThreads / kWave)));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == TRLK_F32)
        filter_bwd_kernel<TRLK_F32><<<grid, kScanThreads, 0, st>>>(a);
    else if (dtype == TRLK_BF16)
        filter_bwd_kernel<TRLK_BF16><<<grid, kScanThreads, 0, st>>>(a);
    else
        filter_bwd_kernel<TRLK_F16><<<grid, kScanThreads, 0, st>>>(a);
    return launch_status("filtered_logps backward");
}
