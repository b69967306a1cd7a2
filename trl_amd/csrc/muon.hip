// K11: updates brought near the nearest matrix with orthonormal rows (or columns) by Newton-Schulz products, for many matrices in one
// call, alone or inside of an optimiser's step.
//
//   u = m' = momentum m + (1 - momentum) g,   with nesterov  u = momentum m' + (1 - momentum) g
//   X = u / max(|u|, eps)   (Frobenius norm; X is u or its transpose, m x n with m <= n)
//   `steps` times:  A = X X^T,  B = b A + c A A,  X = a X + B X
//   p = p (1 - lr decay) - lr stretch X
//
// Bound by the matrix cores: m^2 n + m^3 + 2 m^2 n operations a step (X X^T and A A are symmetric, half of their tiles are computed and
// written twice).  The products run on fp16 operands with fp32 sums.  X is held as two fp16 pieces, x = hi + lo, 22 bits, in units of 2^-14 (its
// singular values stay under 1.3, so do its entries; the units keep what is 2^-28 of the largest out of fp16's subnormals), A and B in
// units of 2^-13.  Results, and steps on parameters in fp32: A and B have two pieces, too, and every product is three, lo hi + hi lo + hi hi, which is fp32's
// precision at a third of the rate (1e-6 of the result).  Steps on parameters in 16 bits: the products take X's hi piece and A and B of one piece, and the term a X, which
// carries the small singular values (they grow by a in each step), all 22 bits but for the last step's.  The largest entries of B are its diagonal's: what their
// rounding leaves is kept in fp32 and multiplied with X's hi piece beside that term (66 rows: 1.96e-3 of the update -> 1.5e-3).  Against the exact
// iteration the update is then off by 0.9 to 1.5e-3 of its size for matrices of independent entries, up to 1.9e-3 where few singular values are large, and where
// entries are alike but for their sign, whose roundings go one way, by up to 1e-2 (ones of 383 x 4096 9.5e-3, an identity 7.7e-3); a parameter in 16 bits, rounded to 2^-9 of
// ITS size and moved by a small part of that, does not show it.  More steps, or other coefficients, whose slopes would make more of the loss take two pieces, too (error_growth).  With one
// piece for X as well those losses were up to 4e-2, with bf16 operands 3e-1.
#include <math.h>

#include <algorithm>
#include <exception>
#include <mutex>
#include <vector>

#include "common.hpp"
#include "gemm_tile.hpp"

namespace trlk {
namespace {

typedef u32x4 u32x4_u __attribute__((aligned(2)));  // vectors at any element alignment
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));

constexpr int kThreads = 256;
constexpr int kChunk = 8192;       // entries of a workgroup of the momentum's pass
constexpr int kTurn = 64;          // rows and columns of a tile of the pass that makes X
constexpr float kUnitX = 16384.f, kUnitA = 8192.f;  // X and A, B are held times these
constexpr int64_t kMostRows = 32768, kMostCols = int64_t(1) << 22, kMostEntries = int64_t(1) << 34;
constexpr size_t kGroupBytes = size_t(1) << 33;  // of workspace, unless one matrix needs more

// One matrix of a launch: X is m x n, m <= n, rows of npad entries, mpad of them (multiples of the k step; what lies between is zero).
struct Mat {
    uint16_t* x;     // narrow ones: partial sums of G, then T.  Others: [2 buffers][hi, lo][mpad][npad], then A and B, [pieces][mpad][mpad] each
    void* p;         // parameter, or the output
    const void* g;   // gradient, or the input
    float* momentum;  // null: no step, the output is X
    const float* d_lr;
    int32_t m, n, mpad, npad;
    float lr, stretch, weight_decay, beta, rest;  // rest: 1 - beta
    int32_t nesterov, tall, pieces;               // tall: p is n x m
    uint32_t first_chunk, first_turn, first_half[3], first_tile[3];  // pieces of the kinds of launches
    __device__ __forceinline__ int64_t plane() const { return int64_t(mpad) * npad; }
    __device__ __forceinline__ int64_t square() const { return int64_t(mpad) * mpad; }
    __device__ __forceinline__ uint16_t* buffer(int i) const { return x + 2 * i * plane(); }
    __device__ __forceinline__ uint16_t* a() const { return x + 4 * plane(); }
    __device__ __forceinline__ uint16_t* b() const { return x + 4 * plane() + pieces * square(); }
    __device__ __forceinline__ float* rest_of_b() const { return reinterpret_cast<float*>(b() + square()); }  // (one piece)
};

// A pointer into global memory.  One that comes from a table in memory may point anywhere, for all that the compiler knows: its loads would be flat ones, and
// whoever uses one would wait for all loads in flight.
template <typename T>
__device__ __forceinline__ T* global(T* p) {
    typedef __attribute__((address_space(1))) T* Global;
    return (T*)(Global)reinterpret_cast<uint64_t>(p);
}
__device__ __forceinline__ Mat mat_at(const Mat* mats, int i) {
    Mat e = mats[i];
    e.x = global(e.x);
    e.p = global(static_cast<char*>(e.p));
    e.g = global(static_cast<const char*>(e.g));
    e.momentum = e.momentum ? global(e.momentum) : nullptr;
    e.d_lr = e.d_lr ? global(e.d_lr) : nullptr;
    return e;
}

constexpr int kTable = 34;
struct MatTable {
    Mat e[kTable];
    Mat* to;
    int32_t n;
};
static_assert(sizeof(MatTable) <= 4096, "a launch's arguments");

__global__ __launch_bounds__(64) void table_kernel(MatTable t) {
    for (int i = threadIdx.x; i < t.n; i += 64) t.to[i] = t.e[i];
}

// The matrix of piece w, all lanes of the wave at it: 64 places at a time, two loads one after the other for up to 4096 matrices
// (a search by halves, eight for 224 adapters: their two passes 30.5 and 29.5 us, so 28.6 and 28.4).
template <typename F>
__device__ __forceinline__ int mat_of(const Mat* e, int n, uint32_t w, F first) {
    const int lane = threadIdx.x & (kWave - 1);
    int lo = 0, left = n;  // it is one of lo .. lo + left - 1
    while (left > 1) {
        const int step = (left + kWave - 1) / kWave, i = lane * step;
        const uint64_t upto = __ballot(i < left && first(e[lo + min(i, left - 1)]) <= w);
        const int k = (__popcll(upto) - 1) * step;
        lo += k;
        left = min(step, left - k);
    }
    return lo;
}
struct FirstChunk {
    __device__ __forceinline__ uint32_t operator()(const Mat& e) const { return e.first_chunk; }
};
struct FirstTurn {
    __device__ __forceinline__ uint32_t operator()(const Mat& e) const { return e.first_turn; }
};

// ---- momentum, norms, X ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float moved(float was, float g, const Mat& e) { return fmaf(e.beta, was, e.rest * g); }
__device__ __forceinline__ float update_of(float now, float g, const Mat& e) { return e.nesterov ? fmaf(e.beta, now, e.rest * g) : now; }

__device__ __forceinline__ void load8f(const float* p, float (&x)[8]) {
    Elem<TRLK_F32>::unpack(*reinterpret_cast<const u32x4_u*>(p), x);
    Elem<TRLK_F32>::unpack(*reinterpret_cast<const u32x4_u*>(p + 4), x + 4);
}
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::type* p, float (&x)[8]) {
#pragma unroll
    for (int k = 0; k < 8; k += Elem<DT>::EPV) Elem<DT>::unpack(*reinterpret_cast<const u32x4_u*>(p + k), x + k);
}

// The momentum moves on; partial sums of u's squares, in 64 bits.
template <int DT>
__global__ __launch_bounds__(kThreads) void momentum_kernel(const Mat* mats, int n_mats, double* partial) {
    __shared__ double scratch[kThreads / kWave];
    const Mat e = mat_at(mats, mat_of(mats, n_mats, blockIdx.x, FirstChunk{}));
    const int64_t numel = int64_t(e.m) * e.n, begin = int64_t(blockIdx.x - e.first_chunk) * kChunk;
    const auto* g = static_cast<const typename Elem<DT>::type*>(e.g);
    double s = 0.0;
    for (int64_t at = begin + threadIdx.x * 8; at < begin + kChunk && at < numel; at += kThreads * 8) {
        float x[8], w[8];
        if (at + 8 <= numel) {
            load8<DT>(g + at, x);
            if (e.momentum) {
                load8f(e.momentum + at, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    w[k] = moved(w[k], x[k], e);
                    x[k] = update_of(w[k], x[k], e);
                }
                *reinterpret_cast<u32x4_u*>(e.momentum + at) = Elem<TRLK_F32>::pack(w);
                *reinterpret_cast<u32x4_u*>(e.momentum + at + 4) = Elem<TRLK_F32>::pack(w + 4);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) s = __builtin_fma(double(x[k]), double(x[k]), s);
        } else {
            for (int64_t k = at; k < numel; ++k) {
                float u = Elem<DT>::load1(g + k);
                if (e.momentum) {
                    const float now = moved(e.momentum[k], u, e);
                    e.momentum[k] = now;
                    u = update_of(now, u, e);
                }
                s = __builtin_fma(double(u), double(u), s);
            }
        }
    }
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double r = 0.0;
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) r += scratch[w];
        partial[blockIdx.x] = r;
    }
}

// kUnitX / max(|u|, eps) of each matrix (NaN where the norm is)
__global__ __launch_bounds__(kThreads) void norm_kernel(const Mat* mats, const double* partial, float* factor, double eps) {
    __shared__ double scratch[kThreads / kWave];
    const Mat& e = mats[blockIdx.x];
    const int64_t n = (int64_t(e.m) * e.n + kChunk - 1) / kChunk;
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) s += partial[e.first_chunk + i];
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    double r = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) r += scratch[w];
    const double norm = sqrt(r);
    factor[blockIdx.x] = float(double(kUnitX) / (norm < eps ? eps : norm));
}

// The value as it stands in a register.  Without this the compiler rounds the same expression to fp16 in two ways, once from its fp32 value and
// once, in one instruction, from its exact one; now and then they differ by a step, and hi and lo did not belong together (fp32 matrices came
// out 10 to 100 times less exact).
__device__ __forceinline__ float settled(float x) {
    asm("" : "+v"(x));
    return x;
}
// x = hi + lo, the rounding of hi made good by lo
__device__ __forceinline__ void split(float x, float& hi, float& lo) {
    x = settled(x);
    hi = float(_Float16(x));
    lo = x - hi;
}
__device__ __forceinline__ void split4(f32x4 x, f32x4& hi, f32x4& lo) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float h, l;
        split(x[k], h, l);
        hi[k] = h;
        lo[k] = l;
    }
}
__device__ __forceinline__ void store_pieces8(uint16_t* hi, int64_t lo_plane, const float (&x)[8]) {
    float h[8], l[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) split(x[k], h[k], l[k]);
    *reinterpret_cast<u32x4*>(hi) = Elem<TRLK_F16>::pack(h);
    *reinterpret_cast<u32x4*>(hi + lo_plane) = Elem<TRLK_F16>::pack(l);
}

// X in two pieces, a tile of 64 x 64 a workgroup, turned over where the parameter is tall; the zeros around X, A and B.  HBM bound: of a 4096-wide model's
// four layers, 671 M entries of bf16, 1417 us, 4.7 TB/s; the momentum's pass before it 1219, 5.5 TB/s.
template <int DT>
__global__ __launch_bounds__(kThreads) void make_x_kernel(const Mat* mats, int n_mats, const float* factor) {
    __shared__ float tile[kTurn][kTurn + 1];
    const int i = mat_of(mats, n_mats, blockIdx.x, FirstTurn{});
    const Mat e = mat_at(mats, i);
    const float f = factor[i];
    const auto* g = static_cast<const typename Elem<DT>::type*>(e.g);
    const uint32_t t = blockIdx.x - e.first_turn, across = uint32_t(e.npad / kTurn);
    const int r0 = int(t / across) * kTurn, c0 = int(t % across) * kTurn;
    const auto value = [&](int64_t at) {
        const float x = Elem<DT>::load1(g + at);
        return (e.momentum ? update_of(e.momentum[at], x, e) : x) * f;
    };
    // eight neighbours of u, factor and all
    const auto eight = [&](int64_t at, float (&x)[8]) {
        load8<DT>(g + at, x);
        if (e.momentum) {
            float w[8];
            load8f(e.momentum + at, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = update_of(w[k], x[k], e);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= f;
    };
    if (e.tall) {  // u is n x m: its rows are X's columns
#pragma unroll
        for (int q = 0; q < kTurn * kTurn / 8 / kThreads; ++q) {
            const int v = q * kThreads + threadIdx.x, c = v / (kTurn / 8), r = v % (kTurn / 8) * 8;
            const int64_t at = int64_t(c0 + c) * e.m + r0 + r;
            float x[8];
            if (c0 + c < e.n && r0 + r + 8 <= e.m) {
                eight(at, x);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = c0 + c < e.n && r0 + r + k < e.m ? value(at + k) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) tile[r + k][c] = x[k];
        }
        __syncthreads();
    }
    for (int v = threadIdx.x; v < kTurn * kTurn / 8; v += kThreads) {
        const int r = v / (kTurn / 8), c = v % (kTurn / 8) * 8;
        const bool inside = r0 + r < e.m && c0 + c + 8 <= e.n;
        float x[8];
        if (e.tall) {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = tile[r][c + k];
        } else if (inside) {
            eight(int64_t(r0 + r) * e.n + c0 + c, x);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = r0 + r < e.m && c0 + c + k < e.n ? value(int64_t(r0 + r) * e.n + c0 + c + k) : 0.f;
        }
        const int64_t to = int64_t(r0 + r) * e.npad + c0 + c;
        store_pieces8(e.buffer(0) + to, e.plane(), x);
        if (!inside) {  // (the entries of X among them are written later)
            const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            store_pieces8(e.buffer(1) + to, e.plane(), zero);
        }
    }
    if (c0 == 0 && e.m < e.mpad) {
        const int gap = e.mpad - e.m;
        for (int v = threadIdx.x; v < kTurn * gap; v += kThreads) {
            const int64_t to = int64_t(r0 + v / gap) * e.mpad + e.m + v % gap;
            for (int q = 0; q < e.pieces; ++q) e.a()[q * e.square() + to] = e.b()[q * e.square() + to] = 0;
        }
    }
}

// ---- products --------------------------------------------------------------------------------------------------------
enum Stage { kStageA, kStageB, kStageX, kStageLast };

struct ProductArgs {
    const Mat* mats;
    int32_t n, from;  // from: the buffer that holds X
    uint32_t tiles, run;
    int32_t reads_lo, writes_lo;  // whether X, and the next X, have their lo piece (16 bits: the last one has not)
    float a, b, c;
};

// The tiles of all matrices of a launch are numbered one after the other, a matrix's so that 16 or 32 neighbours form a patch of 4 x 4 or 4 x 8, and
// dealt out in runs of neighbours to the XCDs (xcd_piece): those that run on one XCD together share their slabs of the operands through its L2.
// bands of 4 rows, column by column
__device__ __forceinline__ void tile_at(int index, int down, int across, int& tr, int& tc) {
    const int band = index / (4 * across), rest = index - band * 4 * across, rows = min(4, down - 4 * band);
    tc = rest / rows;
    tr = band * 4 + rest - tc * rows;
}
// the same for the tiles on and below the diagonal: band k has 16 k + 10 of them, the bands before it 8 k^2 + 2 k
__device__ __forceinline__ void half_tile_at(int index, int down, int& tr, int& tc) {
    int band = int((sqrtf(float(4 + 32 * index)) - 2.f) * (1.f / 16.f));
    while (8 * (band + 1) * (band + 1) + 2 * (band + 1) <= index) ++band;
    while (8 * band * band + 2 * band > index) --band;
    const int rest = index - 8 * band * band - 2 * band, rows = min(4, down - 4 * band), square = rows * 4 * band;
    if (rest < square) {
        tc = rest / rows;
        tr = 4 * band + rest - tc * rows;
        return;
    }
    const int t = rest - square;  // (0, 0), (1, 0), (1, 1), (2, 0) ...
    const int r = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
    tr = 4 * band + r;
    tc = 4 * band + t - r * (r + 1) / 2;
}

// Two neighbouring blocks of four fp16 a lane (the lane groups of 16 hold one after the other) as eight neighbours a lane: the groups 0 and 2
// get the first block's, 1 and 3 the second's; and back.  Offset of a lane's eight in the 32.
__device__ __forceinline__ int pair_offset(int lane) { return ((lane >> 4) & 1) * 16 + (lane >> 5) * 8; }
__device__ __forceinline__ u32x4 pair_up(u32x2 a, u32x2 b) {
    const auto lo = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
    return u32x4{lo[0], hi[0], lo[1], hi[1]};
}
__device__ __forceinline__ void pair_apart(u32x4 q, u32x2& a, u32x2& b) {
    const auto lo = __builtin_amdgcn_permlane16_swap(q.x, q.z, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(q.y, q.w, false, false);
    a = u32x2{lo[0], hi[0]};
    b = u32x2{lo[1], hi[1]};
}

__device__ __forceinline__ float half_at(const uint16_t* p) { return Elem<TRLK_F16>::load1(p); }
template <int DT>
__device__ __forceinline__ f32x4 unpack4(u32x2 q) {
    float x[4];
    Elem<DT>::unpack2(q.x, x);
    Elem<DT>::unpack2(q.y, x + 2);
    return f32x4{x[0], x[1], x[2], x[3]};
}
template <int DT>
__device__ __forceinline__ u32x2 pack4(f32x4 x) { return u32x2{Elem<DT>::pack2(x[0], x[1]), Elem<DT>::pack2(x[2], x[3])}; }

// Four neighbouring entries of a parameter (or the output), `left` of them inside: p = p decay - size x, or p = x.
template <int DT>
__device__ __forceinline__ void finish4(const Mat& e, int64_t at, int left, f32x4 x, float decay, float size) {
    auto* p = static_cast<typename Elem<DT>::type*>(e.p) + at;
    if (left >= 4) {
        f32x4 was = {0.f, 0.f, 0.f, 0.f};
        if constexpr (DT == TRLK_F32) {
            if (e.momentum) was = __builtin_bit_cast(f32x4, *reinterpret_cast<const u32x4_u*>(p));
        } else {
            if (e.momentum) was = unpack4<DT>(*reinterpret_cast<const u32x2_u*>(p));
        }
        if (e.momentum) {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = fmaf(was[k], decay, -size * x[k]);
        }
        if constexpr (DT == TRLK_F32) *reinterpret_cast<u32x4_u*>(p) = __builtin_bit_cast(u32x4, x);
        else *reinterpret_cast<u32x2_u*>(p) = pack4<DT>(x);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < left) Elem<DT>::store1(p + k, e.momentum ? fmaf(Elem<DT>::load1(p + k), decay, -size * x[k]) : x[k]);
    }
}

// A workgroup's tile of a product.  Big: 256 x 256 with the loop of the lm_head's products, 8 waves.
struct BigTile {
    static constexpr int kRows = BM, kCols = BN, kThreads = kHeadThreads, kWaveRows = WM, kWaveCols = WN, kI = MI, kJ = NI, kLds = 2 * kDenseStage;
    static __device__ __forceinline__ int wave_row(int wave) { return wave_m(wave) * WM; }
    static __device__ __forceinline__ int wave_col(int wave) { return wave_n(wave) * WN; }
    template <bool BKM, bool TURNED, typename Runs>
    static __device__ __forceinline__ void product(const Operand A, int m0, const Operand B, int n0, int K, f32x4 (&acc)[kI][kJ], char* smem, Runs runs) {
        gemm_tile_nt_direct<TRLK_F16, BKM, NoLeftKm, Runs, TURNED>(A, m0, B, n0, K, acc, smem, NoLeftKm{}, runs);
    }
};
// Small: 128 x 128 or 64 x 64, 4 waves of a quarter each, for launches whose big tiles would leave CUs idle: four or sixteen times the tiles with as
// much less work, two on a CU.  Of 128 x 128 the bound is the LDS: a step of 64 k moves 96 KB in and out of it for 512 cycles of MFMAs,
// and takes 0.58 us with one tile on a CU and 0.54 with two (165 and 180 GB/s a CU).  Four stages instead of two, which leave room for one
// tile only, and tiles that come through registers two steps ahead were no faster (0.61 and 0.66 us).  Of 64 x 64 it is the transfers' latency: four stages
// (a step on one bf16 matrix of 1024 x 1024 151 us, with three 154, with two 174).  Layouts are those of the big tile's loop; a k-major stage has 64 k rows
// of 256 or 128 bytes.
template <int SIDE, int STAGES>
struct SmallTileOf {
    static constexpr int kRows = SIDE, kCols = SIDE, kThreads = 256, kWaveRows = SIDE / 2, kWaveCols = SIDE / 2, kI = SIDE / 32, kJ = SIDE / 32;
    static constexpr int kStages = STAGES, kHalf = kRows * kRowBytes, kStage = 2 * kHalf, kLds = kStages * kStage, kLoads = kHalf / 1024 / 4;
    static constexpr int kKmRow = SIDE * 2, kKmUnits = SIDE / 8;  // of a k-major stage: bytes and 16-byte units of a k row
    static __device__ __forceinline__ int wave_row(int wave) { return (wave >> 1) * (SIDE / 2); }
    static __device__ __forceinline__ int wave_col(int wave) { return (wave & 1) * (SIDE / 2); }
    // the unit at physical position u of k row r holds logical unit u ^ km_swizzle(r): the eight k rows that two neighbouring groups of 16 lanes
    // read with a transpose load are spread over all banks (two k rows of 128 bytes lie in the 64 banks side by side)
    static __device__ __forceinline__ int km_swizzle(int r) { return SIDE == 128 ? ((r & 3) << 1) ^ (r & 8) : (r & 2) ^ ((r & 8) >> 1); }
    template <bool BKM, bool TURNED, typename Runs>
    static __device__ __forceinline__ void product(const Operand A, int m0, const Operand B, int n0, int K, f32x4 (&acc)[kI][kJ], char* smem, Runs runs) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const char* abase = reinterpret_cast<const char*>(A.p + int64_t(m0) * A.ld);
        const char* bbase = reinterpret_cast<const char*>(BKM ? B.p + n0 : B.p + int64_t(n0) * B.ld);
        const uint32_t lda = uint32_t(A.ld * 2), ldb = uint32_t(B.ld * 2);
        uint32_t ao[kLoads], bo[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int row = (wave + 4 * j) * 8 + lane / kCpr, kc = lane % kCpr ^ tile_swizzle(row);
            ao[j] = uint32_t(min(row, A.rows - 1 - m0)) * lda + uint32_t(kc * 16);
            bo[j] = uint32_t(min(row, B.rows - 1 - n0)) * ldb + uint32_t(kc * 16);
            if constexpr (BKM) {
                const int at = (wave + 4 * j) * 64 + lane, krow = at / kKmUnits, unit = at % kKmUnits ^ km_swizzle(krow);
                bo[j] = uint32_t(krow) * ldb + uint32_t(unit * 16);
            }
        }
        const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>(smem));
        const auto issue = [&](int kt) {
            const int k0 = kt * BK;
            const char* a = abase + runs.left_plane(k0) + int64_t(runs.inside(k0)) * 2;
            const char* b = bbase + runs.right_plane(k0) + int64_t(runs.inside(k0)) * (BKM ? B.ld * 2 : 2);
            const uint32_t to = lds0 + uint32_t(kt % kStages * kStage + wave * 1024);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                DirectLoader<>::transfer(a, ao[j], to + j * 4096);
                DirectLoader<>::transfer(b, bo[j], to + kHalf + j * 4096);
            }
        };
        const int g = lane >> 4, l15 = lane & 15, wr = wave_row(wave), wc = wave_col(wave);
        const int koff[2] = {(g ^ tile_swizzle(l15)) * 16, ((4 + g) ^ tile_swizzle(l15)) * 16};
        int km[kJ];  // k-major: see the big loop
        if constexpr (BKM) {
#pragma unroll
            for (int j = 0; j < kJ; ++j)
                km[j] = (8 * g + (l15 >> 2)) * kKmRow + (((wc + j * 16) / 8 + ((l15 & 3) >> 1)) ^ km_swizzle(8 * g + (l15 >> 2))) * 16 + (l15 & 1) * 8;
        }
#pragma unroll
        for (int i = 0; i < kI; ++i)
#pragma unroll
            for (int j = 0; j < kJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int nk = K / BK;
        u32x4 a[2][kI], b[2][kJ];  // the fragments of both halves of a step
        const auto read = [&](int kt, int ks) {
            const char* sa = smem + kt % kStages * kStage;
            const char* sb = sa + kHalf;
#pragma unroll
            for (int i = 0; i < kI; ++i) a[ks][i] = *reinterpret_cast<const u32x4*>(sa + (wr + i * 16 + l15) * kRowBytes + koff[ks]);
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                if constexpr (BKM) {
                    const uint32_t at = uint32_t(reinterpret_cast<uintptr_t>(sb)) + km[j] + ks * 32 * kKmRow;
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at + 4 * kKmRow));
                    const u32x2 p = __builtin_bit_cast(u32x2, lo), q = __builtin_bit_cast(u32x2, hi);
                    b[ks][j] = u32x4{p.x, p.y, q.x, q.y};
                } else {
                    b[ks][j] = *reinterpret_cast<const u32x4*>(sb + (wc + j * 16 + l15) * kRowBytes + koff[ks]);
                }
            }
        };
        const auto multiply = [&](int ks) {
#pragma unroll
            for (int i = 0; i < kI; ++i)
#pragma unroll
                for (int j = 0; j < kJ; ++j) acc[i][j] = TURNED ? mfma<TRLK_F16>(b[ks][j], a[ks][i], acc[i][j]) : mfma<TRLK_F16>(a[ks][i], b[ks][j], acc[i][j]);
        };
        // `later` stages may still be on their way; what this wave has asked the LDS for has arrived
        const auto landed = [&](int later) {
            static_assert(kStages >= 2 && kStages <= 4 && 6 * kLoads < 64, "up to three later stages, and what the counter holds");
            if (kStages > 3 && later == 3) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(6 * kLoads) : "memory");
            else if (kStages > 2 && later == 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(4 * kLoads) : "memory");
            else if (later == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * kLoads) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
        };
        for (int kt = 0; kt < kStages && kt < nk; ++kt) issue(kt);
        landed(min(kStages, nk) - 1);
        read(0, 0);
        for (int kt = 0; kt < nk; ++kt) {
            // (the fences keep the reads ahead of the MFMAs that run meanwhile: left to itself the compiler puts each beside its first use)
            read(kt, 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(0);
            __builtin_amdgcn_sched_barrier(0);
            if (kt + 1 < nk) {
                // the next stage is there, and everyone has read this one: it is filled again
                landed(min(kt + kStages - 1, nk - 1) - (kt + 1));
                if (kt + kStages < nk) issue(kt + kStages);
                read(kt + 1, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            multiply(1);
            __builtin_amdgcn_sched_barrier(0);
        }
        // (the caller reuses the LDS)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();
    }
};

typedef SmallTileOf<128, 2> SmallTile;
typedef SmallTileOf<64, 4> TinyTile;

// The transposed part of a symmetric result: a wave's entries (128 or 64 x 64, or 32 x 32) go through LDS of its own, rows of its columns (and 8 of padding against
// bank conflicts), and come back with eight neighbours of the other side a lane, by the transpose loads: lane t of a group of 16 points at the
// 8 bytes with columns 4 (t % 4) .. + 3 of row t / 4 (of 4 rows) and receives column t of those rows.
template <typename Tile>
constexpr int mirror_bytes() { return Tile::kWaveCols * (Tile::kWaveRows + 8) * 2; }
template <typename Tile>
constexpr int product_lds() {
    return Tile::kLds > Tile::kThreads / 64 * mirror_bytes<Tile>() ? Tile::kLds : Tile::kThreads / 64 * mirror_bytes<Tile>();
}
template <typename Tile>
__device__ __forceinline__ void mirror(char* mine, const u32x2 (&q)[Tile::kI][Tile::kJ], uint16_t* out, int64_t ld, int i0, int j0, int most, int lane) {
    constexpr int MI = Tile::kI, NI = Tile::kJ, kMirrorRow = (Tile::kWaveRows + 8) * 2;
    const int l15 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int jj = 0; jj < NI; ++jj)
#pragma unroll
        for (int ii = 0; ii < MI; ++ii)
            *reinterpret_cast<u32x2*>(mine + (jj * 16 + l15) * kMirrorRow + (ii * 16 + g * 4) * 2) = q[ii][jj];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const uint32_t base = uint32_t(reinterpret_cast<uintptr_t>(mine)) + (l15 >> 2) * kMirrorRow + (l15 & 3) * 8;
#pragma unroll
    for (int jj = 0; jj < NI / 2; ++jj) {
#pragma unroll
        for (int ii = 0; ii < MI; ++ii) {
            const uint32_t at = base + (jj * 32 + g * 8) * kMirrorRow + ii * 32;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at + 4 * kMirrorRow));
            const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
            const int i = i0 + ii * 16 + l15, j = j0 + jj * 32 + g * 8;
            if (i < most && j < most) *reinterpret_cast<u32x4*>(out + int64_t(i) * ld + j) = u32x4{a.x, a.y, b.x, b.y};
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// One tile of A, B, the next X or, DT, the parameter.  PIECES: two pieces to every operand (fp32).
template <typename Tile, bool PIECES, int STAGE, int DT>
__global__ __launch_bounds__(Tile::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void product_kernel(
    ProductArgs args) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int MI = Tile::kI, NI = Tile::kJ, BM = Tile::kRows, BN = Tile::kCols;
    constexpr int kWhich = std::is_same_v<Tile, TinyTile> ? 2 : std::is_same_v<Tile, SmallTile> ? 1 : 0;
    typedef std::conditional_t<PIECES, PieceRuns, OneRun> Runs;
    constexpr bool kSquare = STAGE == kStageA || STAGE == kStageB;
    const int64_t piece = xcd_piece(blockIdx.x, args.run);
    if (piece >= args.tiles) return;
    const auto first = [](const Mat& e) { return (kSquare ? e.first_half : e.first_tile)[kWhich]; };
    const Mat e = mat_at(args.mats, mat_of(args.mats, args.n, uint32_t(piece), first));
    const int index = int(uint32_t(piece) - first(e));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wr = Tile::wave_row(wave), wc = Tile::wave_col(wave);
    const uint16_t* x = e.buffer(args.from);
    const int64_t plane = e.plane(), square = e.square();
    const int down = (e.m + BM - 1) / BM;
    f32x4 acc[MI][NI];
    const auto runs = [&](int k, int64_t left, int64_t right) {
        if constexpr (PIECES) return PieceRuns{k, left * 2, right * 2};
        else return OneRun{};
    };
    constexpr int kRuns = PIECES ? 3 : 1;
    int tr, tc;
    if constexpr (kSquare) {
        // tiles on and below the diagonal; an entry has the row of the left operand, i, and the right one's, j
        half_tile_at(index, down, tr, tc);
        const int i0 = tr * BM, j0 = tc * BN;
        const uint16_t* from = STAGE == kStageA ? x : e.a();
        const int k = STAGE == kStageA ? e.npad : e.mpad;
        const Operand q{from, k, e.m};
        const int64_t lo = STAGE == kStageA ? plane : square;
        Tile::template product<false, false, Runs>(q, i0, q, j0, kRuns * k, acc, smem, runs(k, lo, lo));
        uint16_t* out = STAGE == kStageA ? e.a() : e.b();
        const int iw = i0 + wr, jw = j0 + wc;
        if (iw >= e.m || jw >= e.m) return;  // (no barrier follows)
        const bool diagonal = !PIECES && STAGE == kStageB && tr == tc;
        // (neighbours past m, up to mpad, are written as zeros: they are the contraction's padding in the next product)
        u32x2 high[MI][NI], low[PIECES ? MI : 1][PIECES ? NI : 1];
        u32x4 was[2][PIECES ? MI : MI / 2];  // A's entries, a column of blocks ahead
        const auto fetch = [&](int jj) {
            const uint16_t* p = e.a() + int64_t(min(jw + jj * 16 + (lane & 15), e.m - 1)) * e.mpad;
#pragma unroll
            for (int ii = 0; ii < MI; ii += 2) {
                const int at = min(iw + ii * 16 + pair_offset(lane), e.mpad - 8);
                was[jj & 1][ii / 2] = *reinterpret_cast<const u32x4*>(p + at);
                if constexpr (PIECES) was[jj & 1][MI / 2 + ii / 2] = *reinterpret_cast<const u32x4*>(p + square + at);
            }
        };
        if constexpr (STAGE == kStageB) fetch(0);
#pragma unroll
        for (int jj = 0; jj < NI; ++jj) {
            const int j = jw + jj * 16 + (lane & 15);
            const bool live = j < e.m;
            const int64_t row = int64_t(live ? j : 0) * e.mpad;
            if (STAGE == kStageB && jj + 1 < NI) fetch(jj + 1);
#pragma unroll
            for (int ii = 0; ii < MI; ii += 2) {
                const int at = iw + ii * 16 + pair_offset(lane);
                const bool there = live && at < e.mpad;
                u32x2 ah[2], al[2];
                if constexpr (STAGE == kStageB) {
                    pair_apart(was[jj & 1][ii / 2], ah[0], ah[1]);
                    if constexpr (PIECES) pair_apart(was[jj & 1][MI / 2 + ii / 2], al[0], al[1]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int i = iw + (ii + u) * 16 + (lane >> 4) * 4;
                    f32x4 v, h, l;
                    if constexpr (STAGE == kStageA) {
                        v = acc[ii + u][jj] * (kUnitA / (kUnitX * kUnitX));
                    } else {
                        f32x4 w = unpack4<TRLK_F16>(ah[u]);
                        if constexpr (PIECES) w += unpack4<TRLK_F16>(al[u]);
                        v = w * args.b + acc[ii + u][jj] * (args.c / kUnitA);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (i + r >= e.m || !live) v[r] = 0.f;
                    split4(v, h, l);
                    if (diagonal && i <= j && j < i + 4 && live) e.rest_of_b()[j] = j == i ? l[0] : j == i + 1 ? l[1] : j == i + 2 ? l[2] : l[3];
                    high[ii + u][jj] = pack4<TRLK_F16>(h);
                    if constexpr (PIECES) low[ii + u][jj] = pack4<TRLK_F16>(l);
                }
                const u32x4 h8 = pair_up(high[ii][jj], high[ii + 1][jj]);
                if (there) *reinterpret_cast<u32x4*>(out + row + at) = h8;
                if constexpr (PIECES) {
                    const u32x4 l8 = pair_up(low[ii][jj], low[ii + 1][jj]);
                    if (there) *reinterpret_cast<u32x4*>(out + square + row + at) = l8;
                }
            }
        }
        if (tr != tc) {
            char* mine = smem + wave * mirror_bytes<Tile>();
            mirror<Tile>(mine, high, out, e.mpad, iw, jw, e.m, lane);
            if constexpr (PIECES) mirror<Tile>(mine, low, out + square, e.mpad, iw, jw, e.m, lane);
        }
    } else {
        const int across = (e.n + BN - 1) / BN;
        tile_at(index, down, across, tr, tc);
        const int r0 = tr * BM, c0 = tc * BN;
        const Operand bs{e.b(), e.mpad, e.m}, xs{x, e.npad, e.npad};
        const float scale = 1.f / kUnitA;
        float decay = 1.f, size = 0.f;
        if constexpr (STAGE == kStageLast) {
            if (e.momentum) {
                const float lr = e.d_lr ? *e.d_lr : e.lr;
                decay = float(1.0 - double(lr) * double(e.weight_decay));
                size = lr * e.stretch;
            }
            if (e.tall) {  // neighbours are those of a column of X, which is the parameter's row
                Tile::template product<true, false, Runs>(bs, r0, xs, c0, kRuns * e.mpad, acc, smem, runs(e.mpad, square, plane));
#pragma unroll
                for (int jj = 0; jj < NI; ++jj) {
                    const int c = c0 + wc + jj * 16 + (lane & 15);
                    if (c >= e.n) continue;
#pragma unroll
                    for (int ii = 0; ii < MI; ++ii) {
                        const int r = r0 + wr + ii * 16 + (lane >> 4) * 4;
                        if (r >= e.m) continue;
                        f32x4 v;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {  // (rows of X's padding are there)
                            const uint16_t* p = x + int64_t(r + k) * e.npad + c;
                            const float high = half_at(p), low = PIECES || args.reads_lo ? half_at(p + plane) : 0.f;
                            if constexpr (PIECES) v[k] = (high + low) * args.a;
                            else v[k] = high * fmaf(e.rest_of_b()[r + k], scale, args.a) + low * args.a;
                        }
                        finish4<DT>(e, int64_t(c) * e.m + r, e.m - r, (v + acc[ii][jj] * scale) * (1.f / kUnitX), decay, size);
                    }
                }
                return;
            }
        }
        Tile::template product<true, true, Runs>(bs, r0, xs, c0, kRuns * e.mpad, acc, smem, runs(e.mpad, square, plane));
        const int cw = c0 + wc;
        if (cw >= e.npad) return;  // (npad is a multiple of a wave's 64 columns: all of them are there or none)
        uint16_t* out = e.buffer(args.from ^ 1);
        // X's own entries, loaded some rows of blocks ahead: a load cannot pass the stores before it, and each would wait for them
        constexpr int kAhead = MI < 4 ? MI : 4;
        u32x4 own[kAhead][NI];  // of each pair of blocks, hi and lo
        float rest[kAhead];
        const auto row_of = [&](int ii) { return int64_t(min(r0 + wr + ii * 16 + (lane & 15), e.m - 1)) * e.npad + cw + pair_offset(lane); };
        const auto fetch = [&](int ii) {
            const uint16_t* p = x + row_of(ii);
            if constexpr (!PIECES) rest[ii % kAhead] = e.rest_of_b()[min(r0 + wr + ii * 16 + (lane & 15), e.m - 1)];
#pragma unroll
            for (int jj = 0; jj < NI; jj += 2) {
                own[ii % kAhead][jj] = *reinterpret_cast<const u32x4*>(p + jj * 16);
                own[ii % kAhead][jj + 1] = PIECES || args.reads_lo ? *reinterpret_cast<const u32x4*>(p + plane + jj * 16) : u32x4{0u, 0u, 0u, 0u};
            }
        };
#pragma unroll
        for (int ii = 0; ii < kAhead; ++ii) fetch(ii);
#pragma unroll
        for (int ii = 0; ii < MI; ++ii) {
            const int r = r0 + wr + ii * 16 + (lane & 15);
            const bool live = r < e.m;
            f32x4 v[NI];
            const float a_hi = PIECES ? args.a : fmaf(rest[ii % kAhead], scale, args.a);
#pragma unroll
            for (int jj = 0; jj < NI; jj += 2) {
                u32x2 xh[2], xl[2];
                pair_apart(own[ii % kAhead][jj], xh[0], xh[1]);
                pair_apart(own[ii % kAhead][jj + 1], xl[0], xl[1]);
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    v[jj + u] = unpack4<TRLK_F16>(xh[u]) * a_hi + unpack4<TRLK_F16>(xl[u]) * args.a + acc[ii][jj + u] * scale;
            }
            if (ii + kAhead < MI) fetch(ii + kAhead);
            if constexpr (STAGE == kStageLast) {
#pragma unroll
                for (int jj = 0; jj < NI; ++jj) {
                    const int c = cw + jj * 16 + (lane >> 4) * 4;
                    if (live && c < e.n) finish4<DT>(e, int64_t(r) * e.n + c, e.n - c, v[jj] * (1.f / kUnitX), decay, size);
                }
            } else {  // (X's padding is zero, and so is what is made of it)
                const int64_t at = row_of(ii);
#pragma unroll
                for (int jj = 0; jj < NI; jj += 2) {
                    u32x2 h2[2], l2[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f32x4 h, l;
                        split4(v[jj + u], h, l);
                        h2[u] = pack4<TRLK_F16>(h);
                        l2[u] = pack4<TRLK_F16>(l);
                    }
                    const u32x4 h8 = pair_up(h2[0], h2[1]), l8 = pair_up(l2[0], l2[1]);
                    if (live) {
                        *reinterpret_cast<u32x4*>(out + at + jj * 16) = h8;
                        if (PIECES || args.writes_lo) *reinterpret_cast<u32x4*>(out + plane + at + jj * 16) = l8;
                    }
                }
            }
        }
    }
}

// ---- narrow matrices: 64 rows or fewer ------------------------------------------------------------------------------------
// With T = the product of the steps' factors, the result is T X, and both T and every step's X X^T are polynomials of the first one's, G = X X^T, which is
// m x m: X is read once for G and once for T X, the steps are products of m x m matrices in one workgroup's LDS,
//   P = a + b G + c G G,  T = P T,  G = P G P.
// G squares the singular values: what X holds in 24 bits needs 48 in G, so all of this is in 64 bits (fp64 runs at full rate here, and there is
// little of it).  Bound by the memory and by launches, three and the tables instead of the 18 of the larger matrices' way: 224 adapters of rank 16 with
// 9 M entries 93 us, 29 of them G's sums, 10 the steps, 28 T X and the parameters, 17 the tables.
constexpr int kNarrow = 64;          // rows at most
constexpr int kCols = 128;           // columns of u at a time in LDS, and of a workgroup that applies T
constexpr int kSpan = 2 * kCols;     // of one that sums for G
constexpr int kLine = kCols + 1;

// u of `cols` columns from c0 on as fp32, [row][column] (kLine apart), zero outside; MOVE: the momentum moves on (else it has).
template <int DT, int MP, bool MOVE>
__device__ __forceinline__ void load_u(const Mat& e, int c0, float* tile) {
    const auto* g = static_cast<const typename Elem<DT>::type*>(e.g);
    const auto value = [&](int64_t at) {
        const float x = Elem<DT>::load1(g + at);
        if (!e.momentum) return x;
        float now = e.momentum[at];
        if constexpr (MOVE) e.momentum[at] = now = moved(now, x, e);
        return update_of(now, x, e);
    };
    const int cols = min(kCols, e.n - c0);
    const auto four = [&](int64_t at, float (&u)[4]) {
        float x[8], w[4];
        if constexpr (DT == TRLK_F32) {
            Elem<DT>::unpack(*reinterpret_cast<const u32x4_u*>(g + at), x);
        } else {
            const u32x2 q = *reinterpret_cast<const u32x2_u*>(g + at);
            Elem<DT>::unpack2(q.x, x);
            Elem<DT>::unpack2(q.y, x + 2);
        }
        if (e.momentum) {
            Elem<TRLK_F32>::unpack(*reinterpret_cast<const u32x4_u*>(e.momentum + at), w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (MOVE) w[k] = moved(w[k], x[k], e);
                x[k] = update_of(w[k], x[k], e);
            }
            if constexpr (MOVE) *reinterpret_cast<u32x4_u*>(e.momentum + at) = Elem<TRLK_F32>::pack(w);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = x[k];
    };
    if (e.tall) {  // cols * m entries one behind the other
        const int64_t from = int64_t(c0) * e.m;
        const int count = cols * e.m;
        for (int i = threadIdx.x * 4; i < count; i += kThreads * 4) {
            float u[4] = {0.f, 0.f, 0.f, 0.f};
            if (i + 4 <= count) four(from + i, u);
            else
                for (int k = 0; i + k < count; ++k) u[k] = value(from + i + k);
            int c = i / e.m, r = i - c * e.m;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i + k < count) tile[r * kLine + c] = u[k];
                if (++r == e.m) r = 0, ++c;
            }
        }
        for (int i = threadIdx.x; i < MP * kCols; i += kThreads) {
            const int r = i / kCols, c = i % kCols;
            if (r >= e.m || c >= cols) tile[r * kLine + c] = 0.f;
        }
    } else {
        for (int i = threadIdx.x; i < MP * kCols / 4; i += kThreads) {
            const int r = i / (kCols / 4), c = i % (kCols / 4) * 4;
            const int64_t at = int64_t(r) * e.n + c0 + c;
            float u[4] = {0.f, 0.f, 0.f, 0.f};
            if (r < e.m) {
                if (c + 4 <= cols) four(at, u);
                else
                    for (int k = 0; c + k < cols; ++k) u[k] = value(at + k);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) tile[r * kLine + c + k] = u[k];
        }
    }
}

// The sum over a workgroup's columns of u u^T.  A lane has 4 x 4 entries of it; with fewer than 64 rows the lanes share the columns.
template <int DT, int MP>
__global__ __launch_bounds__(kThreads) void gram_kernel(const Mat* mats, int n_mats) {
    constexpr int kBlocks = (MP / 4) * (MP / 4), kSlices = kThreads / kBlocks;
    constexpr int kTileBytes = MP * kLine * 4, kSumBytes = kSlices > 1 ? kSlices * MP * MP * 8 : 0;
    __shared__ __attribute__((aligned(16))) char smem[kTileBytes > kSumBytes ? kTileBytes : kSumBytes];
    float* tile = reinterpret_cast<float*>(smem);
    const Mat e = mat_at(mats, mat_of(mats, n_mats, blockIdx.x, FirstChunk{}));
    const int chunk = int(blockIdx.x - e.first_chunk), slice = threadIdx.x / kBlocks, block = threadIdx.x % kBlocks;
    const int bi = block / (MP / 4) * 4, bj = block % (MP / 4) * 4;
    double sum[4][4] = {};
    for (int c0 = chunk * kSpan; c0 < (chunk + 1) * kSpan && c0 < e.n; c0 += kCols) {
        __syncthreads();
        load_u<DT, MP, true>(e, c0, tile);
        __syncthreads();
        for (int c = slice; c < kCols; c += kSlices) {
            double x[4], y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = tile[(bi + k) * kLine + c], y[k] = tile[(bj + k) * kLine + c];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[i][j] = __builtin_fma(x[i], y[j], sum[i][j]);
        }
    }
    double* out = reinterpret_cast<double*>(e.x) + int64_t(chunk) * MP * MP;
    if constexpr (kSlices == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) out[(bi + i) * MP + bj + j] = sum[i][j];
    } else {
        double* sums = reinterpret_cast<double*>(smem);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[slice * MP * MP + (bi + i) * MP + bj + j] = sum[i][j];
        __syncthreads();
        for (int k = threadIdx.x; k < MP * MP; k += kThreads) {
            double s = 0.0;
#pragma unroll
            for (int q = 0; q < kSlices; ++q) s += sums[q * MP * MP + k];
            out[k] = s;
        }
    }
}

// z = f(x y) for symmetric x, y that commute, MP x MP in LDS; `x` and `z` may be the same.  A lane has a square of entries: 1, 2 x 2 or 4 x 4.
template <int MP, typename F>
__device__ __forceinline__ void square_product(const double* x, const double* y, double* z, F f) {
    constexpr int LD = MP + 1, S = MP / 16;
    const int bi = threadIdx.x / 16 * S, bj = threadIdx.x % 16 * S;
    double sum[S][S] = {};
#pragma unroll 8
    for (int k = 0; k < MP; ++k) {
        double p[S], q[S];
#pragma unroll
        for (int i = 0; i < S; ++i) p[i] = x[(bi + i) * LD + k], q[i] = y[k * LD + bj + i];
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < S; ++j) sum[i][j] = __builtin_fma(p[i], q[j], sum[i][j]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < S; ++j) z[(bi + i) * LD + bj + j] = f(sum[i][j], bi + i, bj + j);
    __syncthreads();
}

// T / max(|u|, eps) of a matrix, behind its partial sums.
template <int MP>
__global__ __launch_bounds__(kThreads) void narrow_steps_kernel(const Mat* mats, int steps, double a, double b, double c, double eps) {
    constexpr int LD = MP + 1;
    extern __shared__ double buffers[];
    double *G = buffers, *P = G + MP * LD, *T = P + MP * LD, *W = T + MP * LD;
    const Mat e = mat_at(mats, blockIdx.x);
    const int chunks = (e.n + kSpan - 1) / kSpan;
    double* parts = reinterpret_cast<double*>(e.x);
    for (int k = threadIdx.x; k < MP * MP; k += kThreads) {
        double s = 0.0;
        for (int q = 0; q < chunks; q += 8) {  // (eight loads in flight, added in order)
            double x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = q + u < chunks ? parts[int64_t(q + u) * MP * MP + k] : 0.0;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += x[u];
        }
        G[k / MP * LD + k % MP] = s;
    }
    __syncthreads();
    double trace = 0.0;
    for (int k = 0; k < MP; ++k) trace += G[k * LD + k];
    const double norm = sqrt(trace), f = 1.0 / (norm < eps ? eps : norm);
    __syncthreads();
    for (int k = threadIdx.x; k < MP * LD; k += kThreads) G[k] *= f * f;  // (the last column is nobody's)
    __syncthreads();
    // The rounding of G's sums, some 2^-50 of its trace, takes eigenvalues of zero either way, and one below zero has no way back: it grows by a^2 a step and from
    // size one on by its square (a matrix of rank one: 1e8 too large after 18 steps, NaN after 20).  2^-46 of the trace, more where more partial sums are
    // added up, lifts all of them above zero; an eigenvalue s^2 of the matrix's own moves by less than the rounding of its entries to fp32 moves it.
    if (threadIdx.x < MP) G[threadIdx.x * (LD + 1)] += trace * f * f * 0x1p-46 * (1.0 + chunks * 0x1p-10);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        square_product<MP>(G, G, P, [&](double x, int i, int j) { return c * x + b * G[i * LD + j] + (i == j ? a : 0.0); });
        if (s == 0) {
            for (int k = threadIdx.x; k < MP * LD; k += kThreads) T[k] = P[k] * f;
            __syncthreads();
        } else {
            square_product<MP>(T, P, T, [](double x, int, int) { return x; });
        }
        if (s + 1 == steps) break;
        square_product<MP>(P, G, W, [](double x, int, int) { return x; });
        square_product<MP>(W, P, G, [](double x, int, int) { return x; });
    }
    double* out = parts + int64_t(chunks) * MP * MP;
    for (int k = threadIdx.x; k < MP * MP; k += kThreads) out[k] = T[k / MP * LD + k % MP];
}

// T u for a workgroup's columns, a lane half of a column's entries, and the parameter.
template <int DT, int MP>
__global__ __launch_bounds__(kThreads) void narrow_apply_kernel(const Mat* mats, int n_mats) {
    static_assert(kThreads == 2 * kCols, "two lanes a column");
    __shared__ float tile[MP * kLine];
    const Mat e = mat_at(mats, mat_of(mats, n_mats, blockIdx.x, FirstTurn{}));
    const int c0 = int(blockIdx.x - e.first_turn) * kCols, c = threadIdx.x % kCols;
    const int half = __builtin_amdgcn_readfirstlane(threadIdx.x / kCols);
    const double* T = reinterpret_cast<const double*>(e.x) + int64_t((e.n + kSpan - 1) / kSpan) * MP * MP + half * (MP / 2) * MP;
    float decay = 1.f, size = 0.f;
    if (e.momentum) {
        const float lr = e.d_lr ? *e.d_lr : e.lr;
        decay = float(1.0 - double(lr) * double(e.weight_decay));
        size = lr * e.stretch;
    }
    load_u<DT, MP, false>(e, c0, tile);
    __syncthreads();
    double u[MP];
#pragma unroll
    for (int k = 0; k < MP; ++k) u[k] = tile[k * kLine + c];
    __syncthreads();
#pragma unroll 2
    for (int r = 0; r < MP / 2; ++r) {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < MP; ++k) s = __builtin_fma(T[r * MP + k], u[k], s);
        tile[(half * (MP / 2) + r) * kLine + c] = float(s);
    }
    __syncthreads();
    const int cols = min(kCols, e.n - c0);
    if (e.tall) {
        const int64_t from = int64_t(c0) * e.m;
        const int count = cols * e.m;
        for (int i = threadIdx.x * 4; i < count; i += kThreads * 4) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            int q = i / e.m, r = i - q * e.m;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i + k < count) x[k] = tile[r * kLine + q];
                if (++r == e.m) r = 0, ++q;
            }
            finish4<DT>(e, from + i, count - i, x, decay, size);
        }
    } else {
        for (int i = threadIdx.x; i < e.m * (kCols / 4); i += kThreads) {
            const int r = i / (kCols / 4), q = i % (kCols / 4) * 4;
            if (q >= cols) continue;
            f32x4 x;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = tile[r * kLine + q + k];
            finish4<DT>(e, int64_t(r) * e.n + c0 + q, cols - q, x, decay, size);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up_to(int64_t n, int64_t unit) { return ceil_div(n, unit) * unit; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Rows that a narrow matrix is padded to, 0 for the others.
int narrow_rows(const trlk_muon_matrix& x) {
    const int64_t m = std::min(x.rows, x.cols);
    return m <= 16 ? 16 : m <= 32 ? 32 : m <= kNarrow ? 64 : 0;
}
size_t matrix_bytes(const trlk_muon_matrix& x) {
    if (const int mp = narrow_rows(x)) return up256(size_t(ceil_div(std::max(x.rows, x.cols), kSpan) + 1) * mp * mp * sizeof(double));
    const int64_t m = up_to(std::min(x.rows, x.cols), BK), n = up_to(std::max(x.rows, x.cols), BK);
    return up256(size_t(4 * m * n + 4 * m * m) * 2);  // (A and B in two pieces; of one, the rest of B's diagonal, too, lies in the other's place)
}

// Matrices that go through the launches together: of one type, narrow ones of one kind, as many as the workspace's share holds.
struct Group {
    std::vector<int32_t> each;
    int32_t narrow = 0;
    int64_t chunks = 0;  // partial sums of norms
    size_t bytes = 0;
    size_t total() const { return up256(each.size() * sizeof(Mat)) + up256(each.size() * sizeof(float)) + up256(size_t(chunks) * sizeof(double)) + bytes; }
};
std::vector<Group> groups_of(const trlk_muon_matrix* x, int32_t n) {
    constexpr int kTypes = 3, kKinds = 4;  // fp32, bf16, fp16; matrices of any size and the three narrow kinds
    std::vector<int32_t> each[kTypes * kKinds];
    for (int32_t i = 0; i < n; ++i) {
        if (x[i].rows == 0 || x[i].cols == 0) continue;
        const int type = x[i].dtype == TRLK_F32 ? 0 : x[i].dtype == TRLK_BF16 ? 1 : 2, rows = narrow_rows(x[i]);
        each[type * kKinds + (rows == 0 ? 0 : rows == 16 ? 1 : rows == 32 ? 2 : 3)].push_back(i);
    }
    // (the longest contractions first, so that a launch's last workgroups are short ones)
    for (int type = 0; type < kTypes; ++type) {
        std::vector<int32_t>& order = each[type * kKinds];
        std::stable_sort(order.begin(), order.end(), [&](int32_t i, int32_t j) {
            const int64_t mi = std::min(x[i].rows, x[i].cols), mj = std::min(x[j].rows, x[j].cols), ni = std::max(x[i].rows, x[i].cols), nj = std::max(x[j].rows, x[j].cols);
            return ni != nj ? ni > nj : mi > mj;
        });
    }
    std::vector<Group> groups;
    for (const std::vector<int32_t>& order : each) {
        bool fresh = true;
        for (const int32_t i : order) {
            const size_t need = matrix_bytes(x[i]);
            if (fresh || groups.back().bytes + need > kGroupBytes) {
                groups.emplace_back();
                groups.back().narrow = narrow_rows(x[i]);
                groups.back().each.reserve(order.size());
            }
            fresh = false;
            Group& g = groups.back();
            g.each.push_back(i);
            g.chunks += g.narrow ? 0 : ceil_div(x[i].rows * x[i].cols, kChunk);
            g.bytes += need;
        }
    }
    return groups;
}

size_t most_bytes(const std::vector<Group>& groups) {
    size_t most = 0;
    for (const Group& g : groups) most = std::max(most, g.total());
    return most;
}

int reserve_lds(const void* kernel, int bytes, const char* what) {
    struct Done {
        const void* kernel;
        int device;
    };
    static std::mutex guard;
    static std::vector<Done>& done = *new std::vector<Done>;  // (never destroyed)
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess) device = 0;
    std::lock_guard<std::mutex> lock(guard);
    for (const Done& d : done)
        if (d.kernel == kernel && d.device == device) return TRLK_OK;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail(int(e), "%s: cannot reserve %d bytes of LDS: %s", what, bytes, hipGetErrorString(e));
    done.push_back(Done{kernel, device});
    return TRLK_OK;
}

template <typename Tile, bool PIECES, int STAGE, int DT>
int launch_tiles(ProductArgs a, int64_t tiles, hipStream_t stream, const char* what) {
    const auto kernel = product_kernel<Tile, PIECES, STAGE, DT>;
    constexpr int kBytes = product_lds<Tile>();
    if (const int rc = reserve_lds(reinterpret_cast<const void*>(kernel), kBytes, what)) return rc;
    // runs of 16 tiles, of fewer where an XCD would get under 8 of them, and the same number for all
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(16, tiles / 64)), rounds = ceil_div(tiles, 8 * want);
    a.tiles = uint32_t(tiles);
    a.run = uint32_t(ceil_div(tiles, 8 * rounds));
    kernel<<<xcd_grid(tiles, a.run), Tile::kThreads, kBytes, stream>>>(a);
    return TRLK_OK;
}
// The size of tiles whose launch is done soonest, in units of a big tile's time.  A round is 256 big ones.  Of 128 x 128 two run on a CU, 512 take 0.6 of
// that, 256 or fewer 0.36; of 64 x 64 two, too, 512 take 0.27, 256 or fewer 0.235.  Both sides in us: a step on one bf16 matrix
// of 1024 x 1024 478 with 256 alone, 252 with 128, 150 with 64; 1408 x 1408 314 with 128, 212 with 64; 2048 x 2048 420 and 455, 432 with 64 for
// the symmetric products only, 528 tiles; 8 of 512 x 512 189 and 154; fp32, 24 of 1150 x 2816: X X^T 468 with 256, 431 with 128, A A 222 and 195, X's own
// product, 1320 tiles of 256, 660 and 697.
template <bool PIECES, int STAGE, int DT = TRLK_F32>
int launch_product(const ProductArgs& a, const int64_t (&tiles)[3], hipStream_t stream, const char* what) {
    const double big = double(ceil_div(tiles[0], 256)), small = tiles[1] <= 256 ? 0.36 : 0.6 * double(ceil_div(tiles[1], 512));
    const double tiny = tiles[2] <= 256 ? 0.235 : 0.27 * double(ceil_div(tiles[2], 512));
    if (tiny < small && tiny < big) return launch_tiles<TinyTile, PIECES, STAGE, DT>(a, tiles[2], stream, what);
    if (small < big)
        return launch_tiles<SmallTile, PIECES, STAGE, DT>(a, tiles[1], stream, what);
    return launch_tiles<BigTile, PIECES, STAGE, DT>(a, tiles[0], stream, what);
}

struct Numbers {
    int32_t steps;
    double a, b, c, eps;
};

template <int DT, int MP>
int run_narrow(const Mat* mats, int n, int64_t chunks, int64_t turns, const Numbers& num, hipStream_t stream, const char* what) {
    constexpr int kBytes = 4 * MP * (MP + 1) * 8;
    if (const int rc = reserve_lds(reinterpret_cast<const void*>(narrow_steps_kernel<MP>), kBytes, what)) return rc;
    gram_kernel<DT, MP><<<unsigned(chunks), kThreads, 0, stream>>>(mats, n);
    narrow_steps_kernel<MP><<<unsigned(n), kThreads, kBytes, stream>>>(mats, num.steps, num.a, num.b, num.c, num.eps);
    narrow_apply_kernel<DT, MP><<<unsigned(turns), kThreads, 0, stream>>>(mats, n);
    return TRLK_OK;
}

template <int DT, bool PIECES>
int run_group(const Group& group, const trlk_muon_matrix* x, const trlk_muon_group* groups, const Numbers& num, char* ws, hipStream_t stream, const char* what) {
    const int n = int(group.each.size());
    Mat* mats = reinterpret_cast<Mat*>(ws);
    float* factor = reinterpret_cast<float*>(ws + up256(n * sizeof(Mat)));
    double* partial = reinterpret_cast<double*>(reinterpret_cast<char*>(factor) + up256(n * sizeof(float)));
    char* at = reinterpret_cast<char*>(partial) + up256(size_t(group.chunks) * sizeof(double));
    int64_t chunks = 0, turns = 0, halves[3] = {0, 0, 0}, tiles[3] = {0, 0, 0};
    MatTable t;
    t.n = 0;
    t.to = mats;
    for (int i = 0; i < n; ++i) {
        const trlk_muon_matrix& y = x[group.each[i]];
        Mat& e = t.e[t.n++];
        e = {};
        e.x = reinterpret_cast<uint16_t*>(at);
        at += matrix_bytes(y);
        e.p = y.d_param, e.g = y.d_grad, e.momentum = y.d_momentum;
        e.tall = y.rows > y.cols;
        e.m = int32_t(std::min(y.rows, y.cols)), e.n = int32_t(std::max(y.rows, y.cols));
        e.mpad = int32_t(up_to(e.m, BK)), e.npad = int32_t(up_to(e.n, BK));
        e.pieces = PIECES ? 2 : 1;
        if (groups) {
            const trlk_muon_group& g = groups[y.group];
            e.lr = float(g.lr), e.d_lr = g.d_lr, e.weight_decay = float(g.weight_decay);
            e.beta = float(g.momentum), e.rest = float(1.0 - g.momentum), e.nesterov = g.nesterov;
            const double ratio = double(y.rows) / double(y.cols);
            e.stretch = float(g.adjust == TRLK_MUON_MATCH_ADAMW ? 0.2 * sqrt(double(e.n)) : sqrt(ratio > 1.0 ? ratio : 1.0));
        }
        e.first_chunk = uint32_t(chunks), e.first_turn = uint32_t(turns);
        chunks += group.narrow ? ceil_div(e.n, kSpan) : ceil_div(int64_t(e.m) * e.n, kChunk);
        turns += group.narrow ? ceil_div(e.n, kCols) : int64_t(e.mpad / kTurn) * (e.npad / kTurn);
        for (int k = 0; k < 3; ++k) {
            const int64_t side = k == 2 ? TinyTile::kRows : k == 1 ? SmallTile::kRows : BigTile::kRows, down = ceil_div(e.m, side);
            e.first_half[k] = uint32_t(halves[k]), e.first_tile[k] = uint32_t(tiles[k]);
            halves[k] += down * (down + 1) / 2;
            tiles[k] += down * ceil_div(e.n, side);
        }
        if (t.n == kTable || i + 1 == n) {
            table_kernel<<<1, 64, 0, stream>>>(t);
            t.to += t.n;
            t.n = 0;
        }
    }
    if (group.narrow == 16) return run_narrow<DT, 16>(mats, n, chunks, turns, num, stream, what);
    if (group.narrow == 32) return run_narrow<DT, 32>(mats, n, chunks, turns, num, stream, what);
    if (group.narrow == 64) return run_narrow<DT, 64>(mats, n, chunks, turns, num, stream, what);
    momentum_kernel<DT><<<unsigned(chunks), kThreads, 0, stream>>>(mats, n, partial);
    norm_kernel<<<unsigned(n), kThreads, 0, stream>>>(mats, partial, factor, num.eps);
    make_x_kernel<DT><<<unsigned(turns), kThreads, 0, stream>>>(mats, n, factor);
    ProductArgs a{mats, n, 0, 0, 1, 1, 1, float(num.a), float(num.b), float(num.c)};
    for (int s = 0; s < num.steps; ++s) {
        a.reads_lo = s == 0 || s + 1 < num.steps;
        a.writes_lo = s + 2 < num.steps;
        if (const int rc = launch_product<PIECES, kStageA>(a, halves, stream, what)) return rc;
        if (const int rc = launch_product<PIECES, kStageB>(a, halves, stream, what)) return rc;
        const int rc = s + 1 < num.steps ? launch_product<PIECES, kStageX>(a, tiles, stream, what)
                                         : launch_product<PIECES, kStageLast, DT>(a, tiles, stream, what);
        if (rc) return rc;
        a.from ^= 1;
    }
    return TRLK_OK;
}

// The largest |a s + b s^3 + c s^5| for s in [0, top].
double largest_image(double top, double a, double b, double c) {
    const auto p = [&](double s) { return fabs(s * (a + s * s * (b + c * s * s))); };
    double most = p(top);
    // a + 3 b t + 5 c t^2 = 0, t = s^2
    double roots[2];
    int n = 0;
    if (c != 0.0) {
        const double d = 9.0 * b * b - 20.0 * a * c;
        if (d >= 0.0)
            for (double sign : {-1.0, 1.0}) roots[n++] = (-3.0 * b + sign * sqrt(d)) / (10.0 * c);
    } else if (b != 0.0) {
        roots[n++] = -a / (3.0 * b);
    }
    for (int i = 0; i < n; ++i)
        if (roots[i] > 0.0 && roots[i] < top * top) most = std::max(most, p(sqrt(roots[i])));
    return most;
}

// How far a relative error of one, made in b A + c A A of every step, has grown by the end (or before), for the singular value where that is most: each step
// multiplies what is there by its polynomial's slope.  88 for five steps with the usual coefficients, 930 for ten of them, 870 for five with (4.0848, -6.8946, 2.9270),
// under 2 for coefficients that converge.
constexpr double kMostGrowth = 90.0;  // that one piece may have
double error_growth(const Numbers& num) {
    double most = 0.0;
    for (int i = 1; i <= 64; ++i) {
        double s = i / 64.0, off = 0.0;
        for (int k = 0; k < num.steps && off <= kMostGrowth; ++k) {
            const double t = s * s;
            off = fabs(num.a + t * (3.0 * num.b + t * 5.0 * num.c)) * off + fabs(s * t) * (fabs(num.b) + fabs(num.c) * t);
            s *= num.a + t * (num.b + t * num.c);
        }
        most = std::max(most, off);
    }
    return most;
}

int check_numbers(const Numbers& num, const char* what) {
    TRLK_REQUIRE(num.steps >= 1 && num.steps <= 100, TRLK_ERR_BAD_VALUE, "%s: 1 to 100 steps, not %d", what, num.steps);
    TRLK_REQUIRE(num.eps >= 1e-30 && num.eps <= 1.0, TRLK_ERR_BAD_VALUE, "%s: eps must be in [1e-30, 1]", what);
    TRLK_REQUIRE(isfinite(num.a) && isfinite(num.b) && isfinite(num.c), TRLK_ERR_BAD_VALUE, "%s: coefficients must be finite", what);
    // the fp16 pieces hold singular values up to 65504 / kUnitX, and A and B up to 65504 / kUnitA
    double top = 1.0;
    for (int s = 0; s < num.steps; ++s) {
        const double t = top * top, peak = num.c != 0.0 ? -num.b / (2.0 * num.c) : -1.0;
        double b_most = fabs(num.b * t + num.c * t * t);
        if (peak > 0.0 && peak < t) b_most = std::max(b_most, fabs(num.b * peak + num.c * peak * peak));
        TRLK_REQUIRE(top <= 2.5 && b_most <= 7.0, TRLK_ERR_BAD_VALUE, "%s: with these coefficients singular values grow to %g in step %d", what, top, s);
        top = largest_image(top, num.a, num.b, num.c);
    }
    TRLK_REQUIRE(top <= 1e6, TRLK_ERR_BAD_VALUE, "%s: with these coefficients singular values grow to %g", what, top);
    return TRLK_OK;
}

bool size_ok(const trlk_muon_matrix& y) {
    return y.rows >= 0 && y.cols >= 0 && std::min(y.rows, y.cols) <= kMostRows && std::max(y.rows, y.cols) <= kMostCols && y.rows * y.cols <= kMostEntries;
}
int check_matrices(const trlk_muon_matrix* x, int32_t n, const trlk_muon_group* g, int32_t n_groups, bool step, const char* what) {
    TRLK_REQUIRE(n >= 0 && (n == 0 || x), TRLK_ERR_NULL_POINTER, "%s: null table", what);
    TRLK_REQUIRE(!step || (n_groups >= 0 && (n == 0 || g)), TRLK_ERR_NULL_POINTER, "%s: null groups", what);
    for (int32_t i = 0; step && i < n_groups; ++i) {
        TRLK_REQUIRE(g[i].momentum >= 0.0 && g[i].momentum < 1.0, TRLK_ERR_BAD_VALUE, "%s: momentum must be in [0, 1)", what);
        TRLK_REQUIRE(g[i].weight_decay >= 0.0 && (g[i].d_lr || g[i].lr >= 0.0), TRLK_ERR_BAD_VALUE, "%s: lr and weight_decay must not be negative", what);
        TRLK_REQUIRE(g[i].adjust == TRLK_MUON_ORIGINAL || g[i].adjust == TRLK_MUON_MATCH_ADAMW, TRLK_ERR_BAD_VALUE, "%s: unknown adjustment %d", what, g[i].adjust);
    }
    for (int32_t i = 0; i < n; ++i) {
        const trlk_muon_matrix& y = x[i];
        TRLK_REQUIRE(size_ok(y), TRLK_ERR_BAD_SHAPE, "%s: matrix %d is %lld x %lld", what, i, (long long)y.rows, (long long)y.cols);
        TRLK_REQUIRE(y.dtype == TRLK_F32 || y.dtype == TRLK_BF16 || y.dtype == TRLK_F16, TRLK_ERR_BAD_DTYPE, "%s: matrix %d: unsupported dtype %d", what, i, y.dtype);
        TRLK_REQUIRE(!step || (y.group >= 0 && y.group < n_groups), TRLK_ERR_BAD_VALUE, "%s: matrix %d is in no group", what, i);
        if (y.rows == 0 || y.cols == 0) continue;
        TRLK_REQUIRE(y.d_param && y.d_grad && (y.d_momentum || !step), TRLK_ERR_NULL_POINTER, "%s: matrix %d: null operand", what, i);
        TRLK_REQUIRE(step || !y.d_momentum, TRLK_ERR_BAD_VALUE, "%s: matrix %d has a momentum", what, i);
        TRLK_REQUIRE(aligned_to(y.d_param, elem_size(y.dtype)) && aligned_to(y.d_grad, elem_size(y.dtype)) && aligned_to(y.d_momentum, 4), TRLK_ERR_BAD_STRIDE,
                     "%s: matrix %d: misaligned operand", what, i);
    }
    return TRLK_OK;
}

int run(const trlk_muon_matrix* x, int32_t n, const trlk_muon_group* groups, int32_t n_groups, bool step, const Numbers& num, void* d_workspace,
        size_t workspace_bytes, trlk_stream_t stream_, const char* what) {
    if (const int rc = check_matrices(x, n, groups, n_groups, step, what)) return rc;
    if (const int rc = check_numbers(num, what)) return rc;
    const std::vector<Group> all = groups_of(x, n);
    const size_t need = most_bytes(all);
    if (need == 0) return TRLK_OK;
    TRLK_REQUIRE(d_workspace && workspace_bytes >= need, TRLK_ERR_WORKSPACE, "%s: workspace too small", what);
    TRLK_REQUIRE(aligned_to(d_workspace, 256), TRLK_ERR_WORKSPACE, "%s: misaligned workspace", what);
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    char* ws = static_cast<char*>(d_workspace);
    // (a result shows what one piece loses, a step's parameter of 16 bits does not, unless the loss grows)
    const bool one_piece = step && error_growth(num) <= kMostGrowth;
    for (const Group& g : all) {
        const int dtype = x[g.each[0]].dtype;
        const trlk_muon_group* hyper = step ? groups : nullptr;
        const int rc = dtype == TRLK_F32    ? run_group<TRLK_F32, true>(g, x, hyper, num, ws, stream, what)
                       : dtype == TRLK_BF16 ? (one_piece ? run_group<TRLK_BF16, false> : run_group<TRLK_BF16, true>)(g, x, hyper, num, ws, stream, what)
                                            : (one_piece ? run_group<TRLK_F16, false> : run_group<TRLK_F16, true>)(g, x, hyper, num, ws, stream, what);
        if (rc) return rc;
    }
    return launch_status(what);
}

// (the tables are vectors: what they throw ends here)
template <typename F>
int guarded(const char* what, F f) {
    clear_error();
    try {
        return f();
    } catch (const std::exception& e) {
        return fail(TRLK_ERR_BAD_VALUE, "%s: %s", what, e.what());
    }
}

}  // namespace
}  // namespace trlk

using namespace trlk;

extern "C" size_t trlk_muon_workspace_bytes(const trlk_muon_matrix* matrices, int32_t n_matrices) {
    if (!matrices || n_matrices <= 0) return 0;
    for (int32_t i = 0; i < n_matrices; ++i)
        if (!size_ok(matrices[i])) return 0;
    size_t most = 0;
    guarded("muon", [&] {
        most = most_bytes(groups_of(matrices, n_matrices));
        return TRLK_OK;
    });
    return most;
}

extern "C" int trlk_orthogonalize(const trlk_muon_matrix* matrices, int32_t n_matrices, int32_t steps, double a, double b, double c, double eps,
                                  void* d_workspace, size_t workspace_bytes, trlk_stream_t stream) {
    return guarded("orthogonalize", [&] {
        return run(matrices, n_matrices, nullptr, 0, false, Numbers{steps, a, b, c, eps}, d_workspace, workspace_bytes, stream, "orthogonalize");
    });
}

extern "C" int trlk_muon_step(const trlk_muon_matrix* matrices, int32_t n_matrices, const trlk_muon_group* groups, int32_t n_groups, int32_t steps,
                              double a, double b, double c, double eps, void* d_workspace, size_t workspace_bytes, trlk_stream_t stream) {
    return guarded("muon", [&] {
        return run(matrices, n_matrices, groups, n_groups, true, Numbers{steps, a, b, c, eps}, d_workspace, workspace_bytes, stream, "muon");
    });
}
