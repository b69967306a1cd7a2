// K10: rows of the embedding table times a scale, and the table's gradient.
//
//   out[t, :] = scale * W[ids[t], :]                                   (rounded once)
//   dW[v, :] (+)= scale * sum over t with ids[t] = v of g[t, :]        (fp32 sums, rounded once)
//
// HBM bound: the forward reads n ids and rows and writes n rows, the gradient reads n rows and writes the table, or, where it adds
// to a gradient that is there, reads and writes the rows that occur.  Atomics would make the sums' order, and their last bits, a
// matter of chance, and in 16 bits round at every addition.  So the tokens are sorted by id (a stable radix sort of (id, position)
// pairs, 9 bits a pass at most): the rows of one id are neighbours in the order of their positions, one wave adds them up in
// registers and writes the table's row once.  1000 tokens into a table of 50257 x 1150 in fp16 28 us, 32768 into one of 151936 x 4096 in bf16 301 (192 of
// them the table's zeros, at 6.5 TB/s); added, 8192 into one of 256000 x 2048 38.
#include <algorithm>
#include <atomic>

#include "common.hpp"

namespace trlk {
namespace {

typedef u32x4 u32x4_u __attribute__((aligned(2)));  // a 16-byte vector at any element alignment

constexpr int kThreads = 256;
constexpr int kUnroll = 4;                               // vectors of a thread of the forward
constexpr int kItems = kThreads * kUnroll;
constexpr int64_t kMaxGroups = (int64_t(1) << 32) / 1024 - 1;  // of a launch, whatever its block: it has fewer than 2^32 threads
constexpr int64_t kCacheBytes = int64_t(256) << 20;  // of the last cache
constexpr int64_t kMaxTokens = (int64_t(1) << 31) - 1, kMaxVocab = (int64_t(1) << 31) - 2, kMaxCols = int64_t(1) << 20;

// ids of 32 or 64 bits
struct Ids {
    const void* p;
    int is64;
    __device__ __forceinline__ int64_t at(int64_t i) const {
        return is64 ? static_cast<const int64_t*>(p)[i] : int64_t(static_cast<const int32_t*>(p)[i]);
    }
};

__device__ __forceinline__ void flag_index(int32_t* flag) {
    if (flag) atomicOr(flag, TRLK_FLAG_INDEX_OUT_OF_RANGE);
}

// ---- forward ---------------------------------------------------------------------------------------------------------
struct LookupArgs {
    const void* weight;
    void* out;
    Ids ids;
    int64_t n, vocab, ld;   // ld: entries between two rows of the table
    int32_t cols, vecs;     // vecs: 16-byte vectors of a row, the last one may be cut
    uint64_t magic;         // ceil(2^32 / vecs): divides what is under 2^11 where vecs < kItems
    float scale;
    int32_t* flag;
};

template <int DT>
__device__ __forceinline__ u32x4 scaled(u32x4 q, float scale) {
    float x[Elem<DT>::EPV];
    Elem<DT>::unpack(q, x);
#pragma unroll
    for (int k = 0; k < Elem<DT>::EPV; ++k) x[k] *= scale;
    return Elem<DT>::pack(x);
}

// A workgroup's vectors are consecutive ones of the output, whatever rows they belong to: four loads of a lane are in flight.  PAST: stores past the
// caches, for outputs that with the rows they are read from would not stay there (32768 rows of 4096 in bf16 64 us instead of 75).
template <int DT, bool PAST>
__global__ __launch_bounds__(kThreads) void lookup_kernel(LookupArgs a) {
    typedef typename Elem<DT>::type T;
    constexpr int EPV = Elem<DT>::EPV;
    const T* w = static_cast<const T*>(a.weight);
    T* out = static_cast<T*>(a.out);
    const int64_t total = a.n * a.vecs;
    for (int64_t base = int64_t(blockIdx.x) * kItems; base < total; base += int64_t(gridDim.x) * kItems) {
        const int64_t row0 = base / a.vecs;
        const uint32_t rem = uint32_t(base - row0 * a.vecs);
        int64_t id[kUnroll], row[kUnroll];
        uint32_t col[kUnroll];
        bool live[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const uint32_t at = rem + uint32_t(j * kThreads + threadIdx.x);
            live[j] = base + j * kThreads + threadIdx.x < total;
            uint32_t q;
            if (a.vecs >= kItems) q = at >= uint32_t(a.vecs) ? 1u : 0u;
            else q = uint32_t((uint64_t(at) * a.magic) >> 32);
            row[j] = row0 + q;
            col[j] = (at - q * uint32_t(a.vecs)) * EPV;
            id[j] = live[j] ? a.ids.at(row[j]) : 0;
        }
        u32x4 v[kUnroll];
        bool whole[kUnroll], known[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            known[j] = uint64_t(id[j]) < uint64_t(a.vocab);
            whole[j] = int(col[j]) + EPV <= a.cols;
            if (live[j] && known[j] && whole[j]) v[j] = *reinterpret_cast<const u32x4_u*>(w + id[j] * a.ld + col[j]);
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (!live[j]) continue;
            T* to = out + row[j] * a.cols + col[j];
            if (!known[j]) {
                if (col[j] == 0) flag_index(a.flag);
                const int n = min(EPV, a.cols - int(col[j]));
                for (int k = 0; k < n; ++k) Elem<DT>::store1(to + k, __builtin_nanf(""));
            } else if (whole[j]) {
                const u32x4 q = scaled<DT>(v[j], a.scale);
                if constexpr (PAST) __builtin_nontemporal_store(q, reinterpret_cast<u32x4_u*>(to));
                else *reinterpret_cast<u32x4_u*>(to) = q;
            } else {
                const T* from = w + id[j] * a.ld + col[j];
                for (int k = 0; int(col[j]) + k < a.cols; ++k) Elem<DT>::store1(to + k, Elem<DT>::load1(from + k) * a.scale);
            }
        }
    }
}

// ---- tokens in the order of their ids -----------------------------------------------------------------------------------
// A token that counts for nothing (padding, an id outside the table) gets the key `vocab`, which sorts behind all others.
struct KeyArgs {
    Ids ids;
    int64_t vocab, padding;
    int32_t* flag;
    __device__ __forceinline__ uint32_t key(int64_t i) const {
        const int64_t id = ids.at(i);
        if (uint64_t(id) >= uint64_t(vocab)) {
            flag_index(flag);
            return uint32_t(vocab);
        }
        return id == padding ? uint32_t(vocab) : uint32_t(id);
    }
};

constexpr int kMaxDigit = 9, kBins = 1 << kMaxDigit;  // bits of a pass
constexpr int kSortRows = 4;                          // tokens of a lane: a wave's ranks take 0.5 us a row
constexpr int kSortWaves = kThreads / kWave;
constexpr int kSortTile = kThreads * kSortRows;       // of a workgroup; a wave takes consecutive ones

struct SortArgs {
    KeyArgs source;                 // of the first pass
    const uint32_t *in_key, *in_at;  // of the others
    uint32_t *out_key, *out_at;
    uint32_t* counts;  // [bins][tiles]
    uint32_t n, tiles;
    int32_t shift, bits;
};

// Lanes of the wave with the same digit, as a mask.
__device__ __forceinline__ uint64_t peers(uint32_t digit, int bits) {
    uint32_t lo = ~0u, hi = ~0u;
#pragma unroll
    for (int b = 0; b < kMaxDigit; ++b) {
        if (b < bits) {  // (uniform)
            const uint32_t one = uint32_t(int32_t(digit << (31 - b)) >> 31);  // the bit in all places
            const uint64_t ones = __ballot(one != 0u);
            lo &= ~(uint32_t(ones) ^ one);
            hi &= ~(uint32_t(ones >> 32) ^ one);
        }
    }
    return uint64_t(hi) << 32 | lo;
}

// Ranks of a wave's tokens (kSortRows rows of 64, in order) among those of the wave with the same digit; `count` (LDS, the wave's
// own, zeroed) ends up as the wave's histogram.
__device__ __forceinline__ void wave_ranks(const uint32_t (&key)[kSortRows], int shift, int bits, uint32_t n_rows, uint32_t last,
                                           volatile uint16_t* count, uint32_t (&rank)[kSortRows]) {
    const int lane = threadIdx.x & (kWave - 1);
    const uint32_t low = (1u << bits) - 1u;
#pragma unroll
    for (int r = 0; r < kSortRows; ++r) {
        if (uint32_t(r) < n_rows) {  // (uniform in the wave)
            const bool live = uint32_t(r * kWave + lane) < last;
            const uint32_t digit = (key[r] >> shift) & low;
            const uint64_t same = peers(digit, bits) & __ballot(live);
            const uint16_t before = count[digit];
            __builtin_amdgcn_wave_barrier();
            rank[r] = before + uint32_t(__popcll(same & ((uint64_t(1) << lane) - 1)));
            if (live && (same >> lane) == 1) count[digit] = uint16_t(before + __popcll(same));  // (the last of them)
            __builtin_amdgcn_wave_barrier();
        }
    }
}

template <bool FIRST>
__device__ __forceinline__ uint32_t load_keys(const SortArgs& a, uint32_t begin, uint32_t (&key)[kSortRows], uint32_t (&at)[kSortRows]) {
    const uint32_t lane = threadIdx.x & (kWave - 1), left = begin < a.n ? a.n - begin : 0u;
#pragma unroll
    for (int r = 0; r < kSortRows; ++r) {
        const uint32_t i = r * kWave + lane;
        key[r] = at[r] = 0;
        if (i < left) {
            key[r] = FIRST ? a.source.key(begin + i) : a.in_key[begin + i];
            at[r] = FIRST ? begin + i : a.in_at[begin + i];
        }
    }
    return left;
}

template <bool FIRST>
__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortArgs a) {
    __shared__ uint32_t bins[kBins];
    const int n_bins = 1 << a.bits;
    for (int b = threadIdx.x; b < n_bins; b += kThreads) bins[b] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * kSortTile, left = a.n - begin;
#pragma unroll
    for (int r = 0; r < kSortRows; ++r) {
        const uint32_t i = r * kThreads + threadIdx.x;
        if (i < left) atomicAdd(&bins[((FIRST ? a.source.key(begin + i) : a.in_key[begin + i]) >> a.shift) & (n_bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < n_bins; b += kThreads) a.counts[uint32_t(b) * a.tiles + blockIdx.x] = bins[b];
}

// Exclusive sums of the counts, digit by digit and tile by tile, in place, by one workgroup; a lane takes 16 neighbours (32 tiles of 512 counts at a time
// 10.4 us with 4).
constexpr int kScanThreads = 1024, kScanItems = 16;
__global__ __launch_bounds__(kScanThreads) void sort_scan_kernel(uint32_t* counts, int64_t total) {
    __shared__ uint32_t part[kScanThreads / kWave];
    __shared__ uint32_t carried;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    if (threadIdx.x == 0) carried = 0;
    for (int64_t base = 0; base < total; base += kScanThreads * kScanItems) {
        uint32_t x[kScanItems], sum = 0;
        const int64_t at = base + threadIdx.x * kScanItems;
        const bool whole = at + kScanItems <= total;
#pragma unroll
        for (int k = 0; k < kScanItems; k += 4) {
            if (whole) {
                const u32x4 q = *reinterpret_cast<const u32x4*>(counts + at + k);
                x[k] = q.x, x[k + 1] = q.y, x[k + 2] = q.z, x[k + 3] = q.w;
            } else {
#pragma unroll
                for (int i = k; i < k + 4; ++i) x[i] = at + i < total ? counts[at + i] : 0u;
            }
        }
#pragma unroll
        for (int k = 0; k < kScanItems; ++k) sum += x[k];
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const uint32_t y = __shfl_up(upto, o);
            if (lane >= o) upto += y;
        }
        __syncthreads();  // (the reads of `part` and `carried` before)
        if (lane == kWave - 1) part[wave] = upto;
        __syncthreads();
        uint32_t before = carried + upto - sum;
        for (int w = 0; w < wave; ++w) before += part[w];
#pragma unroll
        for (int k = 0; k < kScanItems; ++k) {
            const uint32_t own = x[k];
            x[k] = before;
            before += own;
        }
#pragma unroll
        for (int k = 0; k < kScanItems; k += 4) {
            if (whole) {
                *reinterpret_cast<u32x4*>(counts + at + k) = u32x4{x[k], x[k + 1], x[k + 2], x[k + 3]};
            } else {
#pragma unroll
                for (int i = k; i < k + 4; ++i)
                    if (at + i < total) counts[at + i] = x[i];
            }
        }
        __syncthreads();
        if (threadIdx.x == kScanThreads - 1) carried = before;
    }
}

template <bool FIRST>
__global__ __launch_bounds__(kThreads) void sort_place_kernel(SortArgs a) {
    __shared__ uint16_t count[kSortWaves][kBins];
    __shared__ uint32_t start[kSortWaves][kBins];
    const int wave = threadIdx.x / kWave, n_bins = 1 << a.bits;
    for (int b = threadIdx.x; b < kSortWaves * kBins; b += kThreads) count[0][b] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * kSortTile + wave * (kSortRows * kWave);
    uint32_t key[kSortRows], at[kSortRows];
    uint32_t rank[kSortRows];
    const uint32_t left = load_keys<FIRST>(a, begin, key, at);
    wave_ranks(key, a.shift, a.bits, (left + kWave - 1) / kWave, left, count[wave], rank);
    __syncthreads();
    for (int b = threadIdx.x; b < n_bins; b += kThreads) {
        uint32_t to = a.counts[uint32_t(b) * a.tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            start[w][b] = to;
            to += count[w][b];
        }
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int r = 0; r < kSortRows; ++r) {
        if (r * kWave + lane < left) {
            const uint32_t to = start[wave][(key[r] >> a.shift) & (n_bins - 1)] + rank[r];
            a.out_key[to] = key[r];
            a.out_at[to] = at[r];
        }
    }
}

// ---- up to 16384 tokens: every token's place is counted ----------------------------------------------------------------------
// A token's place is the number of words (id, position), in 32 bits, that are smaller than its own.  A workgroup holds all words in LDS and counts
// for 32 tokens, 32 lanes each; n^2 comparisons, two instructions, are few for 256 CUs: 8192 tokens 11 us, where one workgroup's radix sort takes 23 and the
// six launches of the kernels above 28 and their gaps (an added gradient of 1024 bf16 columns, us a call, so and by those launches: 2048 tokens 18 and 34, 8192
// 35 and 50, 12000 56 and 62, 16384 64 and 67).
constexpr int kRankThreads = 1024, kRankTokens = 32, kRankSlices = kRankThreads / kRankTokens;
constexpr int64_t kMostRanked = 16384;

struct RankArgs {
    KeyArgs source;
    uint32_t *key, *at;
    uint32_t n;
    int32_t bits;  // of a position
};
constexpr int rank_words(int64_t n) { return int(n + kRankSlices * 4 - 1) / (kRankSlices * 4) * (kRankSlices * 4); }

__global__ __launch_bounds__(kRankThreads) void rank_kernel(RankArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t words[];
    __shared__ uint32_t counts[kRankThreads / kWave][kRankTokens];
    KeyArgs source = a.source;
    if (blockIdx.x != 0) source.flag = nullptr;
    const uint32_t padded = uint32_t(rank_words(a.n));
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < padded; i += kRankThreads) words[i] = i < a.n ? source.key(i) << a.bits | i : ~0u;
    __syncthreads();
    const uint32_t slice = threadIdx.x / kRankTokens, token = blockIdx.x * kRankTokens + threadIdx.x % kRankTokens;
    const uint32_t mine = token < a.n ? words[token] : 0u;
    uint32_t count = 0;
#pragma unroll 4
    for (uint32_t at = slice * 4; at < padded; at += kRankSlices * 4) {
        const u32x4 q = *reinterpret_cast<const u32x4*>(words + at);
        count += q.x < mine;
        count += q.y < mine;
        count += q.z < mine;
        count += q.w < mine;
    }
    count += __shfl_xor(count, kRankTokens);
    if ((threadIdx.x & kRankTokens) == 0) counts[threadIdx.x / kWave][threadIdx.x % kRankTokens] = count;
    __syncthreads();
    if (threadIdx.x >= kRankTokens || token >= a.n) return;
    uint32_t place = 0;
#pragma unroll
    for (int w = 0; w < kRankThreads / kWave; ++w) place += counts[w][threadIdx.x];
    a.key[place] = mine >> a.bits;
    a.at[place] = token;
}

// ---- the table's zeros --------------------------------------------------------------------------------------------------
// 4 KiB a workgroup, past the caches: 1.24 GB 187 us (6.7 TB/s), 0.54 GB 82.  Plain stores 183 and 78, but then what is left in the caches is written back
// under the rows' sums (2000 tokens into 0.54 GB 99 us in all, with plain stores 114; 32768 into 1.24 GB, lookup and all, 374 and 389); four vectors a lane 211
// and 91, workgroups of 1024 196 and 88.
struct ZeroArgs {
    u32x4* p;
    int64_t vecs;
    uint8_t *head, *tail;  // what lies before and behind the whole vectors
    int32_t head_bytes, tail_bytes;
};
__global__ __launch_bounds__(kThreads) void zero_kernel(ZeroArgs z) {
    const u32x4 zero = {0, 0, 0, 0};
    for (int64_t at = int64_t(blockIdx.x) * kThreads + threadIdx.x; at < z.vecs; at += int64_t(gridDim.x) * kThreads) __builtin_nontemporal_store(zero, z.p + at);
    if (blockIdx.x == 0) {
        if (int(threadIdx.x) < z.head_bytes) z.head[threadIdx.x] = 0;
        if (int(threadIdx.x) < z.tail_bytes) z.tail[threadIdx.x] = 0;
    }
}

// ---- the table's gradient ---------------------------------------------------------------------------------------------
constexpr int kChunkBits = 4, kMostLevels = 7;

struct GradArgs {
    const uint32_t *key, *at;  // sorted
    float* part;               // of the chunks of 16, 256 ... places that one id has to itself: their sums [chunk][cols]
    uint32_t first[kMostLevels + 1];  // chunk of each level (from 1 on)
    KeyArgs source;            // (unsorted: direct_kernel)
    const void* g;
    void* dw;
    int64_t ldg, ldw;
    uint32_t n, vocab;
    int32_t cols, levels;
    float scale;
};

// eight consecutive entries
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::type* p, float (&x)[8]) {
#pragma unroll
    for (int k = 0; k < 8; k += Elem<DT>::EPV) Elem<DT>::unpack(*reinterpret_cast<const u32x4_u*>(p + k), x + k);
}
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::type* p, const float (&x)[8]) {
#pragma unroll
    for (int k = 0; k < 8; k += Elem<DT>::EPV) *reinterpret_cast<u32x4_u*>(p + k) = Elem<DT>::pack(x + k);
}

constexpr int kVecs = 4;  // vectors of a lane at most

// A wave's columns: V vectors of 8 a lane, 512 apart.  The row's last vector, where it is cut, is read from 8 before the end and what the one before
// it has, too, is not stored: no lane walks over its rows entry by entry.  (Rows of fewer than 8: NARROW.)
template <int V>
struct Columns {
    int32_t from[V], skip[V];  // skip 8: nothing
    __device__ __forceinline__ Columns(int cols, int first, int lane) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int col = first + v * 512 + lane * 8;
            from[v] = max(0, min(col, cols - 8));
            skip[v] = min(8, max(0, col - max(0, cols - 8)));
        }
    }
};
// eight entries as they lie in memory
template <int DT>
struct Raw {
    u32x4 q[8 / Elem<DT>::EPV];
    template <bool NARROW>
    __device__ __forceinline__ void load(const typename Elem<DT>::type* p, int cols) {
        if constexpr (NARROW) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = k < cols ? Elem<DT>::load1(p + k) : 0.f;
#pragma unroll
            for (int i = 0; i < 8 / Elem<DT>::EPV; ++i) q[i] = Elem<DT>::pack(x + i * Elem<DT>::EPV);
        } else {
#pragma unroll
            for (int i = 0; i < 8 / Elem<DT>::EPV; ++i) q[i] = *reinterpret_cast<const u32x4_u*>(p + i * Elem<DT>::EPV);
        }
    }
    __device__ __forceinline__ void add_to(float (&sum)[8]) const {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8 / Elem<DT>::EPV; ++i) Elem<DT>::unpack(q[i], x + i * Elem<DT>::EPV);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] += x[k];
    }
};

// sum += rows.  AT: row j is p + at[j] * ld, else p + j * ld.
template <int DT, int V, bool NARROW, bool AT>
__device__ __forceinline__ void add_rows(float (&sum)[V][8], uint32_t from, uint32_t to, const uint32_t* at, const void* base, int64_t ld, int cols,
                                         const Columns<V>& c, int lane) {
    constexpr int U = V * (DT == TRLK_F32 ? 2 : 1) >= 8 ? 2 : V * (DT == TRLK_F32 ? 2 : 1) >= 4 ? 4 : 8;  // rows in flight
    const auto* p = static_cast<const typename Elem<DT>::type*>(base);
    for (uint32_t begin = from; begin < to; begin += kWave) {
        const uint32_t count = min(uint32_t(kWave), to - begin);
        uint32_t mine = begin + lane;
        if constexpr (AT) mine = at[min(mine, to - 1)];
        for (uint32_t j = 0; j < count; j += U) {
            Raw<DT> x[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j + u < count) {
                    const auto* row = p + int64_t(uint32_t(__builtin_amdgcn_readlane(mine, j + u))) * ld;
#pragma unroll
                    for (int v = 0; v < V; ++v) x[u][v].template load<NARROW>(row + c.from[v], cols);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j + u < count)
#pragma unroll
                    for (int v = 0; v < V; ++v) x[u][v].add_to(sum[v]);
        }
    }
}

// scale * sum into a row of the table's gradient
template <int ODT, bool ADD, bool NARROW>
__device__ __forceinline__ void finish_row(typename Elem<ODT>::type* row, int from, int skip, int cols, float (&sum)[8], float scale) {
    if (skip >= 8) return;
    auto* out = row + from;
    if (skip == 0 && !NARROW) {
        float was[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if constexpr (ADD) load8<ODT>(out, was);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = ADD ? fmaf(sum[k], scale, was[k]) : sum[k] * scale;
        store8<ODT>(out, sum);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (NARROW ? k < cols : k >= skip) Elem<ODT>::store1(out + k, ADD ? fmaf(sum[k], scale, Elem<ODT>::load1(out + k)) : sum[k] * scale);
    }
}

// Sums of the whole chunks of ids that occur often, a wave each: a token in twenty is the commonest one, image placeholders are most of a batch, and one
// wave would add their rows one after the other.  Level 1 adds up 16 rows, each further one (a launch) 16 chunks of the level before.  Added
// to a table's gradient in fp32: 32768 bf16 rows of 4096, 60 % of them of one id, 637 us with level 1 alone, 175 with two; 2^20 of 1024 24.7 ms, 1.03 with three;
// a token in twenty the commonest 221 and 173 us.
template <int DT, int V, bool NARROW, bool ROWS>
__global__ __launch_bounds__(kThreads) void grad_chunks_kernel(GradArgs a, int level) {
    const int lane = threadIdx.x & (kWave - 1), shift = level * kChunkBits;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave), waves = gridDim.x * (kThreads / kWave);
    const Columns<V> c(a.cols, blockIdx.y * (V * 512), lane);
    for (uint32_t chunk = wave; chunk < a.n >> shift; chunk += waves) {
        const uint32_t from = chunk << shift, to = from + (1u << shift), key = a.key[from];
        if (key >= a.vocab || a.key[to - 1] != key) continue;
        float sum[V][8] = {};
        if constexpr (ROWS) {
            add_rows<DT, V, NARROW, true>(sum, from, to, a.at, a.g, a.ldg, a.cols, c, lane);
        } else {
            const float* before = a.part + int64_t(a.first[level - 1]) * a.cols;
            add_rows<TRLK_F32, V, NARROW, false>(sum, chunk << kChunkBits, (chunk + 1) << kChunkBits, nullptr, before, a.cols, a.cols, c, lane);
        }
        float* part = a.part + int64_t(a.first[level] + chunk) * a.cols;
#pragma unroll
        for (int v = 0; v < V; ++v) finish_row<TRLK_F32, false, NARROW>(part, c.from[v], c.skip[v], a.cols, sum[v], 1.f);
    }
}

// One wave for each sorted place where an id begins (the others are done at once), all of the row's columns in flight: the rows up to the first
// whole chunk, the sums of chunks up to the first whole one of the next level and so on, and down again.
template <int GDT, int ODT, bool ADD, int V, bool NARROW>
__global__ __launch_bounds__(kThreads) void grad_rows_kernel(GradArgs a) {
    const int lane = threadIdx.x & (kWave - 1);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave), waves = gridDim.x * (kThreads / kWave);
    const Columns<V> c(a.cols, blockIdx.y * (V * 512), lane);
    for (uint32_t i = wave; i < a.n; i += waves) {
        // the place before (lane 0), its own and those behind
        const uint32_t place = i + lane;
        const uint32_t seen = place >= 1 && place - 1 < a.n ? a.key[place - 1] : ~0u;
        const uint32_t key = __builtin_amdgcn_readlane(seen, 1);
        if (key >= a.vocab) return;  // (all further ones, too)
        if (uint32_t(__builtin_amdgcn_readlane(seen, 0)) == key) continue;
        uint64_t other = __ballot(seen != key) >> 1;
        uint32_t end = i + (other ? uint32_t(__builtin_ctzll(other)) : kWave - 1);
        // (many of one id, image placeholders for instance: the end is one of the places end .. end + left)
        for (uint32_t left = other ? 0u : a.n - end; left != 0;) {
            const uint32_t step = (left + kWave - 1) / kWave, at = end + min((uint32_t(lane) + 1u) * step, left) - 1u;
            other = __ballot(a.key[at] != key);
            const uint32_t same = other ? uint32_t(__builtin_ctzll(other)) : kWave;  // steps that are this id's to their last place
            end += min(same * step, left);
            left = other ? min(step, a.n - end) - 1u : 0u;
        }
        float sum[V][8] = {};
        const auto whole = [](uint32_t place, int level) { return place >> (level * kChunkBits) << (level * kChunkBits); };
        const auto next = [&](uint32_t place, int level) { return whole(place + (1u << (level * kChunkBits)) - 1u, level); };
        uint32_t to = min(end, next(i, 1));
        add_rows<GDT, V, NARROW, true>(sum, i, to, a.at, a.g, a.ldg, a.cols, c, lane);
        for (int s = 1; s < 2 * a.levels; ++s) {
            const int level = s <= a.levels ? s : 2 * a.levels - s, shift = level * kChunkBits;
            const uint32_t from = to;
            to = max(from, s < a.levels ? min(whole(end, level), next(from, level + 1)) : whole(end, level));
            const float* part = a.part + int64_t(a.first[level]) * a.cols;
            add_rows<TRLK_F32, V, NARROW, false>(sum, from >> shift, to >> shift, nullptr, part, a.cols, a.cols, c, lane);
        }
        add_rows<GDT, V, NARROW, true>(sum, to, end, a.at, a.g, a.ldg, a.cols, c, lane);
        auto* row = static_cast<typename Elem<ODT>::type*>(a.dw) + int64_t(key) * a.ldw;
#pragma unroll
        for (int v = 0; v < V; ++v) finish_row<ODT, ADD, NARROW>(row, c.from[v], c.skip[v], a.cols, sum[v], a.scale);
    }
}

// Up to 1024 tokens need no order: a workgroup for each token looks at all ids, returns if its own occurs before, else lists where it
// occurs and adds those rows up.  One launch: 256 tokens of 1024 columns 6.2 us, 1024 12.6;
// with their places counted first 11.7 and 16.8.
constexpr int64_t kMostDirect = 1024;
template <int GDT, int ODT, bool ADD, bool NARROW>
__global__ __launch_bounds__(kThreads) void grad_direct_kernel(GradArgs a) {
    __shared__ uint32_t list[kMostDirect];
    __shared__ uint32_t counts[kThreads / kWave], before[kThreads / kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t t = blockIdx.x;
    KeyArgs source = a.source;
    if (threadIdx.x != 0 || blockIdx.y != 0) source.flag = nullptr;
    const uint32_t key = source.key(t);
    if (key >= a.vocab) return;
    source.flag = nullptr;
    constexpr int R = kMostDirect / kThreads;
    uint64_t same[R];
    uint32_t count = 0;
    bool earlier = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t i = (wave * R + r) * kWave + lane;
        const bool is = i < a.n && source.key(i) == key;
        same[r] = __ballot(is);
        earlier |= __ballot(is && i < t) != 0;
        count += uint32_t(__popcll(same[r]));
    }
    if (lane == 0) counts[wave] = count, before[wave] = earlier;
    __syncthreads();
    uint32_t at = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
        if (before[w]) return;  // (the same for all)
        if (w < wave) at += counts[w];
        total += counts[w];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (same[r] >> lane & 1) list[at + __popcll(same[r] & ((uint64_t(1) << lane) - 1))] = (wave * R + r) * kWave + lane;
        at += uint32_t(__popcll(same[r]));
    }
    __syncthreads();
    // (a wave's columns are consecutive ones)
    const int from = (blockIdx.y * (kThreads / kWave) + wave) * 512;
    if (from >= a.cols) return;
    const Columns<1> c(a.cols, from, lane);
    float sum[1][8] = {};
    add_rows<GDT, 1, NARROW, true>(sum, 0, total, list, a.g, a.ldg, a.cols, c, lane);
    finish_row<ODT, ADD, NARROW>(static_cast<typename Elem<ODT>::type*>(a.dw) + int64_t(key) * a.ldw, c.from[0], c.skip[0], a.cols, sum[0], a.scale);
}

// ---- host ------------------------------------------------------------------------------------------------------------
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t up16(size_t n) { return (n + 15) / 16 * 16; }
bool known(int dtype) { return dtype == TRLK_F32 || dtype == TRLK_BF16 || dtype == TRLK_F16; }

int key_bits(int64_t vocab) {
    int bits = 1;
    while (bits < 32 && (uint64_t(vocab) >> bits) != 0) ++bits;  // (the keys go up to `vocab`)
    return bits;
}
bool ranked(int64_t n, int64_t vocab) { return n <= kMostRanked && key_bits(vocab) + key_bits(n - 1) <= 32; }

// A further level from 512 chunks on: below, a wave adds them up itself (4096 rows of 4096, 60 % of one id, 98 us).
int levels_of(int64_t n) {
    int levels = 1;
    while (levels < kMostLevels && n >> (levels * kChunkBits) > 512) ++levels;
    return levels;
}
int64_t chunks_of(int64_t n, int levels) {  // of the levels 1 .. levels
    int64_t sum = 0;
    for (int l = 1; l <= levels; ++l) sum += n >> (l * kChunkBits);
    return sum;
}

// The workspace: sorted keys and positions, the many-workgroup sort's second pair and counts, the chunks' sums.
struct Layout {
    size_t each, counts, part, total;
    Layout(int64_t n, int64_t vocab, int64_t cols) {
        each = up16(size_t(n) * 4);
        counts = ranked(n, vocab) ? 0 : 2 * each + up16(size_t(ceil_div(n, kSortTile)) * kBins * 4);
        part = 2 * each + counts;
        total = n <= kMostDirect ? 16 : part + up16(size_t(chunks_of(n, levels_of(n))) * size_t(cols) * 4);
    }
};

ZeroArgs zero_args(void* to, int64_t bytes) {
    ZeroArgs z{};
    char* p = static_cast<char*>(to);
    const int64_t gap = (16 - int64_t(reinterpret_cast<uintptr_t>(p) & 15)) & 15, head = gap < bytes ? gap : bytes;
    z.vecs = (bytes - head) / 16;
    z.p = reinterpret_cast<u32x4*>(p + head);
    z.head = reinterpret_cast<uint8_t*>(p), z.tail = reinterpret_cast<uint8_t*>(p + head + z.vecs * 16);
    z.head_bytes = int32_t(head), z.tail_bytes = int32_t(bytes - head - z.vecs * 16);
    return z;
}
int launch_rank(const RankArgs& a, hipStream_t stream) {
    static std::atomic<uint64_t> reserved{0};  // a bit for each device
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess) device = 0;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (!(reserved.load() & bit)) {
        constexpr int kBytes = rank_words(kMostRanked) * 4;
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(rank_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e != hipSuccess) return fail(int(e), "embedding_bwd: cannot reserve %d bytes of LDS: %s", kBytes, hipGetErrorString(e));
        reserved.fetch_or(bit);
    }
    rank_kernel<<<unsigned(ceil_div(a.n, kRankTokens)), kRankThreads, rank_words(a.n) * 4, stream>>>(a);
    return TRLK_OK;
}

// Sorted keys and positions by many workgroups.
void sort_tokens(const KeyArgs& source, int64_t n, char* ws, const Layout& layout, hipStream_t stream, const uint32_t** keys, const uint32_t** places) {
    uint32_t* buf[2][2];
    for (int i = 0; i < 4; ++i) buf[i / 2][i % 2] = reinterpret_cast<uint32_t*>(ws + i * layout.each);
    const int bits = key_bits(source.vocab), passes = (bits + kMaxDigit - 1) / kMaxDigit, digit = (bits + passes - 1) / passes;
    SortArgs a{};
    a.source = source;
    a.counts = reinterpret_cast<uint32_t*>(ws + 4 * layout.each);
    a.n = uint32_t(n);
    a.tiles = uint32_t(ceil_div(n, kSortTile));
    for (int p = 0; p < passes; ++p) {
        a.shift = p * digit;
        a.bits = digit;
        a.in_key = buf[(p + 1) & 1][0], a.in_at = buf[(p + 1) & 1][1];
        a.out_key = buf[p & 1][0], a.out_at = buf[p & 1][1];
        if (p == 0) sort_count_kernel<true><<<a.tiles, kThreads, 0, stream>>>(a);
        else sort_count_kernel<false><<<a.tiles, kThreads, 0, stream>>>(a);
        sort_scan_kernel<<<1, kScanThreads, 0, stream>>>(a.counts, int64_t(a.tiles) << digit);
        a.source.flag = nullptr;  // (raised while counting)
        if (p == 0) sort_place_kernel<true><<<a.tiles, kThreads, 0, stream>>>(a);
        else sort_place_kernel<false><<<a.tiles, kThreads, 0, stream>>>(a);
    }
    *keys = a.out_key;
    *places = a.out_at;
}

template <int GDT, int ODT, bool ADD, int V, bool NARROW>
void launch_sorted(const GradArgs& a, hipStream_t stream) {
    const int64_t y = ceil_div(a.cols, V * 512), most = kMaxGroups / y, waves = kThreads / kWave;
    const auto grid = [&](int64_t n) { return dim3(unsigned(std::min(ceil_div(n, waves), most)), unsigned(y)); };
    grad_chunks_kernel<GDT, V, NARROW, true><<<grid(a.n >> kChunkBits), kThreads, 0, stream>>>(a, 1);
    for (int l = 2; l <= a.levels; ++l) grad_chunks_kernel<TRLK_F32, V, NARROW, false><<<grid(a.n >> (l * kChunkBits)), kThreads, 0, stream>>>(a, l);
    grad_rows_kernel<GDT, ODT, ADD, V, NARROW><<<grid(a.n), kThreads, 0, stream>>>(a);
}
template <int GDT, int ODT, bool ADD>
void launch_rows(const GradArgs& a, bool direct, hipStream_t stream) {
    if (direct) {
        const dim3 grid(a.n, unsigned(ceil_div(a.cols, kThreads * 8)));
        if (a.cols < 8) grad_direct_kernel<GDT, ODT, ADD, true><<<grid, kThreads, 0, stream>>>(a);
        else grad_direct_kernel<GDT, ODT, ADD, false><<<grid, kThreads, 0, stream>>>(a);
    } else if (a.cols < 8) {
        launch_sorted<GDT, ODT, ADD, 1, true>(a, stream);
    } else if (a.cols <= 512) {
        launch_sorted<GDT, ODT, ADD, 1, false>(a, stream);
    } else if (a.cols <= 1024) {
        launch_sorted<GDT, ODT, ADD, 2, false>(a, stream);
    } else {
        launch_sorted<GDT, ODT, ADD, kVecs, false>(a, stream);
    }
}
template <int GDT, int ODT>
void launch_rows(const GradArgs& a, bool direct, bool add, hipStream_t stream) {
    if (add) launch_rows<GDT, ODT, true>(a, direct, stream);
    else launch_rows<GDT, ODT, false>(a, direct, stream);
}

}  // namespace
}  // namespace trlk

using namespace trlk;

extern "C" int trlk_embedding_fwd(const void* d_weight, int dtype, int64_t vocab, int64_t cols, int64_t row_stride, const void* d_ids,
                                  int32_t id_bits, int64_t n, float scale, void* d_out, int32_t* d_error_flag, trlk_stream_t stream_) {
    clear_error();
    TRLK_REQUIRE(known(dtype), TRLK_ERR_BAD_DTYPE, "embedding: unsupported dtype %d", dtype);
    TRLK_REQUIRE(id_bits == 32 || id_bits == 64, TRLK_ERR_BAD_VALUE, "embedding: ids have 32 or 64 bits, not %d", id_bits);
    TRLK_REQUIRE(n >= 0 && n <= kMaxTokens && vocab >= 0 && vocab <= kMaxVocab && cols >= 0 && cols <= kMaxCols, TRLK_ERR_BAD_SHAPE,
                 "embedding: bad sizes: %lld tokens, table %lld x %lld", (long long)n, (long long)vocab, (long long)cols);
    TRLK_REQUIRE(row_stride >= cols || vocab <= 1, TRLK_ERR_BAD_STRIDE, "embedding: row stride %lld under %lld columns", (long long)row_stride, (long long)cols);
    if (n == 0 || cols == 0) return TRLK_OK;
    TRLK_REQUIRE(d_ids && d_out && (d_weight || vocab == 0), TRLK_ERR_NULL_POINTER, "embedding: null pointer");
    TRLK_REQUIRE(aligned_to(d_weight, elem_size(dtype)) && aligned_to(d_out, elem_size(dtype)) && aligned_to(d_ids, id_bits / 8), TRLK_ERR_BAD_STRIDE,
                 "embedding: misaligned operand");
    LookupArgs a{};
    a.weight = d_weight, a.out = d_out, a.ids = Ids{d_ids, id_bits == 64};
    a.n = n, a.vocab = vocab, a.ld = row_stride, a.cols = int32_t(cols);
    a.vecs = int32_t(ceil_div(cols, dtype == TRLK_F32 ? 4 : 8));
    a.magic = ((uint64_t(1) << 32) + a.vecs - 1) / a.vecs;
    a.scale = scale, a.flag = d_error_flag;
    const int64_t need = ceil_div(n * a.vecs, kItems);
    const unsigned grid = unsigned(need < kMaxGroups ? need : kMaxGroups);
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    const bool past = n * cols * int64_t(elem_size(dtype)) >= kCacheBytes / 2;
    const auto launch = [&](auto plain, auto beyond) { (past ? beyond : plain)<<<grid, kThreads, 0, stream>>>(a); };
    if (dtype == TRLK_F32) launch(lookup_kernel<TRLK_F32, false>, lookup_kernel<TRLK_F32, true>);
    else if (dtype == TRLK_BF16) launch(lookup_kernel<TRLK_BF16, false>, lookup_kernel<TRLK_BF16, true>);
    else launch(lookup_kernel<TRLK_F16, false>, lookup_kernel<TRLK_F16, true>);
    return launch_status("embedding_fwd");
}

extern "C" size_t trlk_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t cols) {
    if (n <= 0 || n > kMaxTokens || vocab < 0 || vocab > kMaxVocab || cols < 0 || cols > kMaxCols) return 0;
    return Layout(n, vocab, cols).total;
}

extern "C" int trlk_embedding_bwd(const void* d_grad, int dtype, int64_t n, int64_t cols, int64_t grad_stride, const void* d_ids, int32_t id_bits,
                                  int64_t vocab, float scale, int64_t padding_idx, int32_t accumulate, void* d_dweight, int out_dtype,
                                  int64_t out_stride, int32_t* d_error_flag, void* d_workspace, size_t workspace_bytes, trlk_stream_t stream_) {
    clear_error();
    TRLK_REQUIRE(known(dtype) && (out_dtype == dtype || out_dtype == TRLK_F32), TRLK_ERR_BAD_DTYPE,
                 "embedding_bwd: gradients of dtype %d into dtype %d (the same, or fp32)", dtype, out_dtype);
    TRLK_REQUIRE(id_bits == 32 || id_bits == 64, TRLK_ERR_BAD_VALUE, "embedding_bwd: ids have 32 or 64 bits, not %d", id_bits);
    TRLK_REQUIRE(n >= 0 && n <= kMaxTokens && vocab >= 0 && vocab <= kMaxVocab && cols >= 0 && cols <= kMaxCols, TRLK_ERR_BAD_SHAPE,
                 "embedding_bwd: bad sizes: %lld tokens, table %lld x %lld", (long long)n, (long long)vocab, (long long)cols);
    TRLK_REQUIRE((grad_stride >= cols || n <= 1) && (accumulate ? out_stride >= cols || vocab <= 1 : out_stride == cols), TRLK_ERR_BAD_STRIDE,
                 "embedding_bwd: bad row strides %lld and %lld for %lld columns", (long long)grad_stride, (long long)out_stride, (long long)cols);
    if (cols == 0 || vocab == 0 || (n == 0 && accumulate)) return TRLK_OK;
    TRLK_REQUIRE(d_dweight && (n == 0 || (d_grad && d_ids)), TRLK_ERR_NULL_POINTER, "embedding_bwd: null pointer");
    TRLK_REQUIRE(aligned_to(d_grad, elem_size(dtype)) && aligned_to(d_dweight, elem_size(out_dtype)) && aligned_to(d_ids, id_bits / 8), TRLK_ERR_BAD_STRIDE,
                 "embedding_bwd: misaligned operand");
    TRLK_REQUIRE(n == 0 || (d_workspace && workspace_bytes >= trlk_embedding_bwd_workspace_bytes(n, vocab, cols) && aligned_to(d_workspace, 16)),
                 TRLK_ERR_WORKSPACE, "embedding_bwd: workspace too small or misaligned");
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    const bool direct = n <= kMostDirect, by_rank = !direct && ranked(n, vocab);
    const KeyArgs source{Ids{d_ids, id_bits == 64}, vocab, padding_idx, d_error_flag};
    const Layout layout(n, vocab, cols);
    char* ws = static_cast<char*>(d_workspace);
    GradArgs a{};
    if (!accumulate) {
        const ZeroArgs z = zero_args(d_dweight, vocab * cols * int64_t(elem_size(out_dtype)));
        const int64_t need = std::max<int64_t>(1, ceil_div(z.vecs, kThreads));
        zero_kernel<<<unsigned(std::min(need, kMaxGroups)), kThreads, 0, stream>>>(z);
    }
    if (n == 0) return launch_status("embedding_bwd");
    if (by_rank) {
        const RankArgs r{source, reinterpret_cast<uint32_t*>(ws), reinterpret_cast<uint32_t*>(ws + layout.each), uint32_t(n), key_bits(n - 1)};
        if (const int rc = launch_rank(r, stream)) return rc;
        a.key = r.key, a.at = r.at;
    } else if (!direct) {
        sort_tokens(source, n, ws, layout, stream, &a.key, &a.at);
    }
    a.source = source;
    a.part = reinterpret_cast<float*>(ws + layout.part);
    a.g = d_grad, a.dw = d_dweight, a.ldg = grad_stride, a.ldw = out_stride;
    a.n = uint32_t(n), a.vocab = uint32_t(vocab), a.cols = int32_t(cols), a.levels = levels_of(n), a.scale = scale;
    for (int l = 1; l <= a.levels; ++l) a.first[l] = uint32_t(chunks_of(n, l - 1));
    const bool add = accumulate != 0;
    if (dtype == TRLK_F32) launch_rows<TRLK_F32, TRLK_F32>(a, direct, add, stream);
    else if (dtype == TRLK_BF16 && out_dtype == TRLK_BF16) launch_rows<TRLK_BF16, TRLK_BF16>(a, direct, add, stream);
    else if (dtype == TRLK_BF16) launch_rows<TRLK_BF16, TRLK_F32>(a, direct, add, stream);
    else if (out_dtype == TRLK_F16) launch_rows<TRLK_F16, TRLK_F16>(a, direct, add, stream);
    else launch_rows<TRLK_F16, TRLK_F32>(a, direct, add, stream);
    return launch_status("embedding_bwd");
}
