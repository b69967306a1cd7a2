// K10: rows of the embedding table times a scale, and the table's gradient.
//
//   out[t, :] = scale * W[ids[t], :]                                   (rounded once)
//   dW[v, :] (+)= scale * sum over t with ids[t] = v of g[t, :]        (fp32 sums, rounded once)
//
// HBM bound: the forward reads n ids and rows and writes n rows, the gradient reads n rows and writes the table, or, where it adds
// to a gradient that is there, reads and writes the rows that occur.  Atomics would make the sums' order, and their last bits, a
// matter of chance, and in 16 bits round at every addition.  So the tokens are sorted by id (a stable radix sort of (id, position)
// pairs, 9 bits a pass at most): the rows of one id are neighbours in the order of their positions, one workgroup adds them up in
// registers and writes the table's row once.
#include "common.hpp"

namespace trlk {
namespace {

typedef u32x4 u32x4_u __attribute__((aligned(2)));  // a 16-byte vector at any element alignment

constexpr int kThreads = 256;
constexpr int kUnroll = 4;                               // vectors of a thread of the forward
constexpr int kItems = kThreads * kUnroll;
constexpr int64_t kMaxGroups = (int64_t(1) << 32) / 1024 - 1;  // of a launch, whatever its block: it has fewer than 2^32 threads
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

// A workgroup's vectors are consecutive ones of the output, whatever rows they belong to: four loads of a lane are in flight.
template <int DT>
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
                *reinterpret_cast<u32x4_u*>(to) = scaled<DT>(v[j], a.scale);
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
constexpr int kSortRows = 16;                         // tokens of a lane
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
    uint64_t mask = ~uint64_t(0);
    for (int b = 0; b < bits; ++b) {
        const bool one = (digit >> b) & 1u;
        const uint64_t ones = __ballot(one);
        mask &= one ? ones : ~ones;
    }
    return mask;
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

// Exclusive sums of the counts, digit by digit and tile by tile, in place.
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* counts, int64_t total) {
    __shared__ uint32_t part[1024 / kWave];
    __shared__ uint32_t carried;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    if (threadIdx.x == 0) carried = 0;
    for (int64_t base = 0; base < total; base += 4096) {
        uint32_t x[4], sum = 0;
        const int64_t at = base + threadIdx.x * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[k] = at + k < total ? counts[at + k] : 0u;
            sum += x[k];
        }
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const uint32_t y = __shfl_up(upto, o);
            if (lane >= o) upto += y;
        }
        __syncthreads();  // (the last round's reads of `part` and `carried`)
        if (lane == kWave - 1) part[wave] = upto;
        __syncthreads();
        uint32_t before = carried + upto - sum;
        for (int w = 0; w < wave; ++w) before += part[w];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (at + k < total) counts[at + k] = before;
            before += x[k];
        }
        __syncthreads();
        if (threadIdx.x == 1023) carried = before;
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

// ---- the table's gradient ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void zero_kernel(u32x4* p, int64_t vecs, uint8_t* tail, int bytes) {
    const u32x4 z = {0, 0, 0, 0};
    const int64_t base = int64_t(blockIdx.x) * kItems + threadIdx.x;
    for (int64_t at = base; at < vecs; at += int64_t(gridDim.x) * kItems) {
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
            if (at + j * kThreads < vecs) __builtin_nontemporal_store(z, p + at + j * kThreads);
    }
    if (blockIdx.x == 0 && int(threadIdx.x) < bytes) tail[threadIdx.x] = 0;
}

struct GradArgs {
    const uint32_t *key, *at;  // sorted
    const void* g;
    void* dw;
    int64_t ldg, ldw;
    uint32_t n, vocab;
    int32_t cols;
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

// One workgroup for each sorted place where an id begins (the others return at once), and for 2048 columns.
template <int GDT, int ODT, bool ADD>
__global__ __launch_bounds__(kThreads) void grad_rows_kernel(GradArgs a) {
    typedef typename Elem<GDT>::type TG;
    typedef typename Elem<ODT>::type TO;
    const int lane = threadIdx.x & (kWave - 1);
    const int col = (blockIdx.y * kThreads + threadIdx.x) * 8;
    for (uint32_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const uint32_t key = a.key[i];
        if (key >= a.vocab) return;  // (all further ones, too)
        if (i > 0 && a.key[i - 1] == key) continue;
        uint32_t end = i + 1;
        while (true) {
            const uint64_t other = __ballot(end + lane >= a.n || a.key[end + lane] != key);
            if (other) {
                end += uint32_t(__builtin_ctzll(other));
                break;
            }
            end += kWave;
        }
        if (col >= a.cols) continue;
        const TG* g = static_cast<const TG*>(a.g) + col;
        TO* out = static_cast<TO*>(a.dw) + int64_t(key) * a.ldw + col;
        float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (col + 8 <= a.cols) {
#pragma unroll 4
            for (uint32_t j = i; j < end; ++j) {
                float x[8];
                load8<GDT>(g + int64_t(a.at[j]) * a.ldg, x);
#pragma unroll
                for (int k = 0; k < 8; ++k) sum[k] += x[k];
            }
            float was[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if constexpr (ADD) load8<ODT>(out, was);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[k] = ADD ? fmaf(sum[k], a.scale, was[k]) : sum[k] * a.scale;
            store8<ODT>(out, sum);
        } else {
            const int left = a.cols - col;
            for (uint32_t j = i; j < end; ++j) {
                const TG* row = g + int64_t(a.at[j]) * a.ldg;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < left) sum[k] += Elem<GDT>::load1(row + k);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < left) Elem<ODT>::store1(out + k, ADD ? fmaf(sum[k], a.scale, Elem<ODT>::load1(out + k)) : sum[k] * a.scale);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t up16(size_t n) { return (n + 15) / 16 * 16; }
bool known(int dtype) { return dtype == TRLK_F32 || dtype == TRLK_BF16 || dtype == TRLK_F16; }

size_t sort_bytes(int64_t n) { return 4 * up16(size_t(n) * 4) + up16(size_t(ceil_div(n, kSortTile)) * kBins * 4); }

// Sorted keys and positions, in the workspace.
void sort_tokens(const KeyArgs& source, int64_t n, char* ws, hipStream_t stream, const uint32_t** keys, const uint32_t** places) {
    const size_t each = up16(size_t(n) * 4);
    uint32_t* buf[2][2];
    for (int i = 0; i < 4; ++i) buf[i / 2][i % 2] = reinterpret_cast<uint32_t*>(ws + i * each);
    int bits = 1;
    while (bits < 32 && (uint64_t(source.vocab) >> bits) != 0) ++bits;  // (the keys go up to `vocab`)
    const int passes = (bits + kMaxDigit - 1) / kMaxDigit, digit = (bits + passes - 1) / passes;
    SortArgs a{};
    a.source = source;
    a.counts = reinterpret_cast<uint32_t*>(ws + 4 * each);
    a.n = uint32_t(n);
    a.tiles = uint32_t(ceil_div(n, kSortTile));
    for (int p = 0; p < passes; ++p) {
        a.shift = p * digit;
        a.bits = digit;
        a.in_key = buf[(p + 1) & 1][0], a.in_at = buf[(p + 1) & 1][1];
        a.out_key = buf[p & 1][0], a.out_at = buf[p & 1][1];
        if (p == 0) sort_count_kernel<true><<<a.tiles, kThreads, 0, stream>>>(a);
        else sort_count_kernel<false><<<a.tiles, kThreads, 0, stream>>>(a);
        sort_scan_kernel<<<1, 1024, 0, stream>>>(a.counts, int64_t(a.tiles) << digit);
        a.source.flag = nullptr;  // (raised while counting)
        if (p == 0) sort_place_kernel<true><<<a.tiles, kThreads, 0, stream>>>(a);
        else sort_place_kernel<false><<<a.tiles, kThreads, 0, stream>>>(a);
    }
    *keys = a.out_key;
    *places = a.out_at;
}

template <int GDT, int ODT>
void launch_rows(const GradArgs& a, bool add, hipStream_t stream) {
    const int64_t y = ceil_div(a.cols, kThreads * 8);
    const int64_t most = kMaxGroups / y;
    const dim3 grid(unsigned(a.n < most ? a.n : most), unsigned(y));
    if (add) grad_rows_kernel<GDT, ODT, true><<<grid, kThreads, 0, stream>>>(a);
    else grad_rows_kernel<GDT, ODT, false><<<grid, kThreads, 0, stream>>>(a);
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
    if (dtype == TRLK_F32) lookup_kernel<TRLK_F32><<<grid, kThreads, 0, stream>>>(a);
    else if (dtype == TRLK_BF16) lookup_kernel<TRLK_BF16><<<grid, kThreads, 0, stream>>>(a);
    else lookup_kernel<TRLK_F16><<<grid, kThreads, 0, stream>>>(a);
    return launch_status("embedding_fwd");
}

extern "C" size_t trlk_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t cols) {
    if (n <= 0 || n > kMaxTokens || vocab < 0 || vocab > kMaxVocab || cols < 0 || cols > kMaxCols) return 0;
    return sort_bytes(n);
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
    if (!accumulate) {
        char* p = static_cast<char*>(d_dweight);
        const int64_t bytes = vocab * cols * int64_t(elem_size(out_dtype));
        // (whole vectors from the first aligned address on; what lies before and behind it goes with the last launch argument)
        const int64_t head = (16 - int64_t(reinterpret_cast<uintptr_t>(p) & 15)) & 15;
        const int64_t first = head < bytes ? head : bytes, vecs = (bytes - first) / 16, tail = bytes - first - vecs * 16;
        if (first) zero_kernel<<<1, kThreads, 0, stream>>>(nullptr, 0, reinterpret_cast<uint8_t*>(p), int(first));
        const int64_t need = ceil_div(vecs, kItems);
        if (vecs || tail)
            zero_kernel<<<unsigned(need < 1 ? 1 : need < kMaxGroups ? need : kMaxGroups), kThreads, 0, stream>>>(
                reinterpret_cast<u32x4*>(p + first), vecs, reinterpret_cast<uint8_t*>(p + first + vecs * 16), int(tail));
    }
    if (n == 0) return launch_status("embedding_bwd");
    GradArgs a{};
    sort_tokens(KeyArgs{Ids{d_ids, id_bits == 64}, vocab, padding_idx, d_error_flag}, n, static_cast<char*>(d_workspace), stream, &a.key, &a.at);
    a.g = d_grad, a.dw = d_dweight, a.ldg = grad_stride, a.ldw = out_stride;
    a.n = uint32_t(n), a.vocab = uint32_t(vocab), a.cols = int32_t(cols), a.scale = scale;
    if (dtype == TRLK_F32) launch_rows<TRLK_F32, TRLK_F32>(a, accumulate != 0, stream);
    else if (dtype == TRLK_BF16 && out_dtype == TRLK_BF16) launch_rows<TRLK_BF16, TRLK_BF16>(a, accumulate != 0, stream);
    else if (dtype == TRLK_BF16) launch_rows<TRLK_BF16, TRLK_F32>(a, accumulate != 0, stream);
    else if (out_dtype == TRLK_F16) launch_rows<TRLK_F16, TRLK_F16>(a, accumulate != 0, stream);
    else launch_rows<TRLK_F16, TRLK_F32>(a, accumulate != 0, stream);
    return launch_status("embedding_bwd");
}
