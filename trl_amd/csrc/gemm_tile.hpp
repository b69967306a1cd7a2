// The tile of the matrix products on the matrix cores: C[256 x 256] += A[256 x K] * B[256 x K]^T, both operands row-major with K
// contiguous, or either of them k-major.  Shared by the lm_head's kernels and the orthogonalised updates.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace trlk {
namespace {

constexpr int BM = 256, BN = 256, BK = 64;  // a workgroup's tile, the k step
constexpr int WGM = 2, WGN = 4;               // waves along M and N
constexpr int kHeadThreads = WGM * WGN * 64;
#define TRLK_HEAD_KERNEL __global__ __launch_bounds__(kHeadThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
constexpr int WM = BM / WGM, WN = BN / WGN;  // per-wave tile
constexpr int MI = WM / 16, NI = WN / 16;    // MFMA blocks of it
constexpr int MB = WM / 32, NB = WN / 32;    // ... in the forward
constexpr int kLdsRow = BK + 8;  // register-staged loop: elements per LDS row (16 bytes of padding keep 16-byte reads conflict-free)
constexpr int kCpr = BK / 8;                        // 16-byte chunks per tile row
constexpr int kRowStep = kHeadThreads / kCpr;       // rows staged per pass of the workgroup
constexpr int kLoadsA = BM / kRowStep, kLoadsB = BN / kRowStep;
constexpr int kTileABytes = BM * kLdsRow * 2, kTileBBytes = BN * kLdsRow * 2;
constexpr int kStageBytes = kTileABytes + kTileBBytes;
constexpr int kRowBytes = BK * 2;                    // direct-to-LDS loop: a dense LDS row
constexpr int kDenseA = BM * kRowBytes, kDenseStage = (BM + BN) * kRowBytes;
static_assert(BM % kRowStep == 0 && BN % kRowStep == 0, "tile shape");

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The 16x16x32 shape reads and writes half as many accumulators per multiply-add as 32x32x16 does.  The part is limited by
// power under matrix load, so that shows as speed: a bare loop of MFMAs on random bf16 operands runs at 2020-2060 TFLOP/s
// (2.05-2.12 GHz) against 1830-1880 TFLOP/s (1.87-1.90 GHz), on zeros both at 2450-2490 TFLOP/s (2.4 GHz).
// The forward uses 32x32x16.  Its loop has registers for two sets of fragments there (nothing of the softmax state is
// spilled) and takes, against the same loop as the products', 272 for 286 us with 1396 tokens, H = 2048, V = 50257 and
// 302 for 330 us with 879 tokens, H = 1024, V = 151665; 8345 for 8240 us with 9664 tokens, H = 3584, V = 151936, where
// power decides, is the other side.  The logits come out the same, to the last bit, in both shapes (180000 compared, bf16
// and fp16, sums that cancel and sums that do not): the backward's recompute may use the other one, and the rounding of z
// still cancels against that in log_z.  But the layout of 16x16x32 spreads a token's exponentials over twice as many lanes,
// which changes the order of THEIR sum and the last bits of log_z; with the forward's loop as it is, what a run has stored of
// its old or its reference policy stays what it computes again.
template <int DT>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == TRLK_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// The same value, but nothing computed from it is kept across loop iterations: what the compiler hoists out of the
// forward's tile loop it spills, and a reload waits for every tile transfer in flight.
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A value that is the same in every lane, in a scalar register.
__device__ __forceinline__ float uniform(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }

template <int DT>
__device__ __forceinline__ f32x16 mfma_fwd(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == TRLK_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// Where a wave sits in the tile.  A SIMD runs waves w and w + 4: they differ in their columns (N) by half the tile, so
// that a tile of at most 128 columns leaves every SIMD one wave with work, not two of them both.
__device__ __forceinline__ int wave_m(int wave) { return (wave >> 1) & 1; }
__device__ __forceinline__ int wave_n(int wave) { return (wave & 1) | ((wave >> 2) << 1); }

// One operand of the NT product: `rows` x K, row-major with leading dimension ld (elements).  The right operand may
// instead be given "k-major" (BKM below): K x `rows`, row-major with leading dimension ld -- the transpose of what the
// product wants, read through the LDS transpose loads; its columns must be readable (and zero) up to the next
// multiple of the tile size.
struct Operand {
    const uint16_t* p;
    int64_t ld;
    int rows;
};
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// The contraction's k as it lies in the operands: one run (the k of the loop is the operands' own), or, for operands that are each the sum
// of two pieces, x = hi + lo, one plane behind the other, three runs of `k` (a multiple of the k step): lo * hi, hi * lo and hi * hi.
// lo * lo is below the rounding of fp32 where a piece has 11 bits.  Bytes to add for the planes, and the k inside of them.
struct OneRun {
    __device__ __forceinline__ int64_t left_plane(int) const { return 0; }
    __device__ __forceinline__ int64_t right_plane(int) const { return 0; }
    __device__ __forceinline__ int inside(int k0) const { return k0; }
};
struct PieceRuns {
    int k;
    int64_t left_lo, right_lo;  // bytes from the hi plane to the lo plane
    __device__ __forceinline__ int64_t left_plane(int k0) const { return k0 < k ? left_lo : 0; }
    __device__ __forceinline__ int64_t right_plane(int k0) const { return k0 >= k && k0 < 2 * k ? right_lo : 0; }
    __device__ __forceinline__ int inside(int k0) const { return k0 < k ? k0 : k0 < 2 * k ? k0 - k : k0 - 2 * k; }
};

// Direct-to-LDS variant of the tile loop (K % BK == 0): `global_load_lds_dwordx4` moves 16 bytes per
// lane from memory straight into LDS, 1 KiB contiguous per wave instruction = 8 tile rows of 64 k, with no register
// staging and no ds_write.  Rows are dense (no padding is possible inside a wave's 1 KiB), so bank conflicts are avoided
// by an XOR swizzle of the 16-byte chunk index: the chunk at physical position pc of row r holds logical chunk
//   pc ^ swz(r),  swz(r) = (r & 7) ^ ((r >> 3) & 1),
// which makes the 16 rows that one ds_read_b128 phase touches cover all 64 banks once.  The lane
// fetches that logical chunk from memory (a permutation inside one row, still coalesced) and the
// fragment reads apply the same XOR.
//
// The loop keeps two 64 KiB stages in LDS; a stage is refilled as soon as the barrier that ends its last use has passed,
// one step before it is needed again.
__device__ __forceinline__ int tile_swizzle(int r) { return (r & 7) ^ ((r >> 3) & 1); }

// Loader side of the direct-to-LDS loop: per-lane source offsets of the wave's tile blocks and the
// transfer of one stage.
// BKM: the right operand is k-major.  Its stage is then 64 k rows of 512 bytes (256 columns); one transfer fills two
// k rows; the 16-byte unit at physical position pu of k row r holds logical unit pu ^ ((r & 3) << 1) ^ (r & 8), which
// spreads the eight k rows that two neighbouring groups of 16 lanes read with a transpose load over all banks.
// LEFT: the left operand travels this way too (otherwise LeftKm moves it).
template <bool BKM = false, bool LEFT = true, typename Runs = OneRun>
struct DirectLoader {
    static constexpr int kWaves = kHeadThreads / 64, kRowsPerBlk = 1024 / kRowBytes;
    static constexpr int kBlkA = LEFT ? BM / kRowsPerBlk / kWaves : 0, kBlkB = BN / kRowsPerBlk / kWaves;  // per wave and stage
    static constexpr int kStageLoads = kBlkA + kBlkB;
    static_assert(BM % (kRowsPerBlk * kWaves) == 0 && BN % (kRowsPerBlk * kWaves) == 0 && BN == 256, "blocks per wave");
    const char *abase, *bbase;
    char* smem;
    int wave;
    int64_t bkstep;  // bytes between two k of the right operand
    uint32_t ao[LEFT ? kBlkA : 1], bo[kBlkB];
    Runs runs;

    __device__ __forceinline__ DirectLoader(const Operand A, int m0, const Operand B, int n0, char* lds, Runs runs_ = {}) : smem(lds), runs(runs_) {
        const int lane = fresh(threadIdx.x & 63);
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: LDS targets stay scalar
        const int rr = lane / kCpr, pc = lane % kCpr;  // row inside a block, chunk position
        abase = reinterpret_cast<const char*>(A.p + int64_t(m0) * A.ld);
        bbase = reinterpret_cast<const char*>(BKM ? B.p + n0 : B.p + int64_t(n0) * B.ld);
        bkstep = BKM ? B.ld * 2 : 2;
        const uint32_t lda = uint32_t(A.ld * 2), ldb = uint32_t(B.ld * 2);  // (a tile spans less than 4 GiB)
#pragma unroll
        for (int j = 0; j < kBlkA; ++j) {
            const int row = (wave + kWaves * j) * kRowsPerBlk + rr;
            const int kc = pc ^ tile_swizzle(row);  // the logical chunk this lane fetches
            const int r = m0 + row < A.rows ? row : A.rows - 1 - m0;
            ao[j] = uint32_t(r) * lda + uint32_t(kc * 16);
        }
#pragma unroll
        for (int j = 0; j < kBlkB; ++j) {
            if constexpr (BKM) {
                const int krow = (wave + kWaves * j) * 2 + (lane >> 5);
                const int lu = (lane & 31) ^ ((krow & 3) << 1) ^ (krow & 8);  // the logical 16-byte unit this lane fetches
                bo[j] = uint32_t(krow) * ldb + uint32_t(lu * 16);
                continue;
            }
            const int row = (wave + kWaves * j) * kRowsPerBlk + rr;
            const int kc = pc ^ tile_swizzle(row);
            const int r = n0 + row < B.rows ? row : B.rows - 1 - n0;
            bo[j] = uint32_t(r) * ldb + uint32_t(kc * 16);
        }
    }
    // One 1 KiB transfer: 16 bytes per lane from `src` to LDS offset `lds` + 16 * lane.  Issued as
    // inline assembly on purpose: the compiler books a global_load_lds as an access of both memory
    // and LDS, after which every wait on a fragment read becomes lgkmcnt(0) (it stalls on the
    // reads just issued); the loop keeps its own vmcnt bookkeeping for these transfers anyway.
    // (m0 is a reserved register; naming it as clobbered is what tells the compiler not to keep a value there)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    // The source is a uniform 64-bit base (scalar registers) plus the lane's 32-bit byte offset: one vector register
    // per transfer instead of an address pair, and the k step is added on the scalar side.
    static __device__ __forceinline__ void transfer(const char* base, uint32_t lane_off, uint32_t lds) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(lane_off),
                     "s"(reinterpret_cast<uint64_t>(base))
                     : "memory", "m0");
    }
#pragma clang diagnostic pop
    __device__ __forceinline__ uint32_t lds_base(int buf) const {
        return uint32_t(reinterpret_cast<uintptr_t>(smem)) + uint32_t(buf * kDenseStage);
    }
    // transfer j of a stage (A blocks first, then B blocks)
    __device__ __forceinline__ void issue_one(int buf, int k0, int j) const {
        if (j < kBlkA)
            transfer(abase + runs.left_plane(k0) + int64_t(runs.inside(k0)) * 2, ao[j], lds_base(buf) + (wave + kWaves * j) * 1024);
        else
            transfer(bbase + runs.right_plane(k0) + int64_t(runs.inside(k0)) * bkstep, bo[j - kBlkA], lds_base(buf) + kDenseA + (wave + kWaves * (j - kBlkA)) * 1024);
    }
    __device__ __forceinline__ void issue(int buf, int k0) const {
#pragma unroll
        for (int j = 0; j < kStageLoads; ++j) issue_one(buf, k0, j);
    }
    // the first two stages of a product; both must be free (all reads of the LDS done)
    __device__ __forceinline__ void prologue(int K) const {
        issue(0, 0);
        if (K > BK) issue(1, BK);
    }
    __device__ __forceinline__ void first_stage_landed(int nk) const {
        if (nk >= 2)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kStageLoads) : "memory");
        else
            __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
};

// The left operand of the dHidden product straight from the weight: k-major (A.p is [krows, A.rows], K = krows rounded up to
// the k step) and, with CONVERT, bf16 that becomes fp16 times a power of two.  A stage is 64 k rows of 256 columns, laid out
// like a k-major right operand's; it goes through registers, because the conversion is done on the way: a lane holds 4 vectors
// of 8 columns, of k rows 16 apart, loaded one step before they are converted and written to the LDS.  k rows beyond the last
// are read as the last (the other operand is zero there), columns beyond the last as the last 8 (nobody stores them).
// The conversion is what this costs beside the plain loop: 1392 tokens, H = 2048, V = 128256, backward of a bf16 problem 1562 us,
// of an fp16 problem (nothing to convert) 1555; behind every MFMA of the refill instead of behind two of three 1577.
// An entry whose scaled value fp16 does not hold counts as fp16's largest (see direct_scale).
template <bool CONVERT>
struct LeftKm {
    static constexpr int kVecs = 4;
    const char* base;
    char* lds;
    uint32_t row_bytes, col;  // (a tile spans less than 4 GiB)
    int row0, krows;
    float scale, top;  // top: the largest magnitude converted so far, times the scale
    __device__ __forceinline__ LeftKm(const Operand A, int m0, int krows_, float scale_, char* smem)
        : krows(krows_), scale(scale_), top(0.f) {
        // FP16_OVFL: what overflows fp16 becomes its largest value (infinities stay), for the rest of the wave's life.  A bit of
        // the mode register, where a clamp would be two instructions more per pair of columns in the tile loop.
        if constexpr (CONVERT) asm volatile("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 23, 1), 1" ::: "memory");
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        base = reinterpret_cast<const char*>(A.p + m0);
        row_bytes = uint32_t(A.ld * 2);
        row0 = wave * 2 + (lane >> 5);
        const int unit = (lane & 31) ^ ((row0 & 3) << 1) ^ (row0 & 8);  // the logical 16-byte unit of this lane, as in DirectLoader
        col = uint32_t(min(unit * 8, A.rows - m0 - 8)) * 2u;
        lds = smem + wave * 1024 + lane * 16;
    }
    __device__ __forceinline__ void load(int k0, int j, u32x4& w) const {
        const int row = min(row0 + 16 * j, krows - 1 - k0);
        w = *reinterpret_cast<const u32x4*>(base + int64_t(k0) * row_bytes + (uint32_t(row) * row_bytes + col));
    }
    // two neighbouring columns; exact wherever fp16 holds the scaled value (below its range one rounding to nearest)
    __device__ __forceinline__ void convert(uint32_t& w) {
        if constexpr (CONVERT) {
            const float lo = __uint_as_float(w << 16) * scale, hi = __uint_as_float(w & 0xffff0000u) * scale;
            asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(top) : "v"(lo), "v"(hi));
            w = Elem<TRLK_F16>::pack2(lo, hi);
        }
    }
    __device__ __forceinline__ void store(int buf, int j, u32x4 w) const {
        *reinterpret_cast<u32x4*>(lds + buf * kDenseStage + j * 8192) = w;
    }
    // the first two stages into the LDS, the third (or, where there is none, the last) into `w`
    __device__ __forceinline__ void prologue(int nk, u32x4 (&w)[kVecs]) {
        u32x4 first[2][kVecs];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < kVecs; ++j) load(min(s, nk - 1) * BK, j, first[s][j]);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t x = first[s][j][i];
                    convert(x);
                    first[s][j][i] = x;
                }
                store(s, j, first[s][j]);
            }
#pragma unroll
        for (int j = 0; j < kVecs; ++j) load(min(2, nk - 1) * BK, j, w[j]);
    }
};
struct NoLeftKm {};

// What a wave whose rows or columns all lie beyond the operands does in place of the tile loop: it moves its share of the
// tiles (exactly the transfers, waits and barriers of the loop) and spends nothing on matrix work.
template <bool BKM, bool LEFT, typename Runs, typename Left = NoLeftKm>
__device__ __forceinline__ void move_tiles_only(const DirectLoader<BKM, LEFT, Runs>& loader, int K, bool prefetched, Left left = {}) {
    const int nk = K / BK;
    u32x4 w[4];
    if (!prefetched) loader.prologue(K);
    if constexpr (LEFT) {
        loader.first_stage_landed(nk);
    } else {
        left.prologue(nk, w);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
#pragma unroll 1
    for (int kt = 0; kt < nk; ++kt) {
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kt + 2 < nk) {
            loader.issue(kt & 1, (kt + 2) * BK);
            if constexpr (!LEFT) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t x = w[j][i];
                        left.convert(x);
                        w[j][i] = x;
                    }
                    left.store(kt & 1, j, w[j]);
                    left.load(min(kt + 3, nk - 1) * BK, j, w[j]);
                }
            }
        }
    }
}

// `left`: a LeftKm, where the left operand is k-major.  TURNED: an accumulator block holds four neighbouring rows of the right operand for one of
// the left operand (acc_turned_...), not the other way round.
template <int DT, bool BKM = false, typename Left = NoLeftKm, typename Runs = OneRun, bool TURNED = false>
__device__ __forceinline__ void gemm_tile_nt_direct(const Operand A, int m0, const Operand B, int n0, int K,
                                                    f32x4 (&acc)[MI][NI], char* smem, Left&& left = {}, Runs runs = {}) {
    constexpr bool AKM = !std::is_same_v<std::decay_t<Left>, NoLeftKm>;
    const DirectLoader<BKM, !AKM, Runs> loader(A, m0, B, n0, smem, runs);
    constexpr int kStageLoads = DirectLoader<BKM, !AKM, Runs>::kStageLoads;
    const int lane = threadIdx.x & 63, wave = loader.wave;
    const int wm = wave_m(wave), wn = wave_n(wave);

    // --- fragment side (blocks start at multiples of 16 rows, so the swizzle depends on the lane only).  A fragment is
    // 16 rows x 32 k: lane l holds the 8 k from 8 (l / 16) on of row l % 16.
    const int g = lane >> 4, l15 = lane & 15;
    const int koff[2] = {(g ^ tile_swizzle(l15)) * 16, ((4 + g) ^ tile_swizzle(l15)) * 16};
    const int fa_row = (wm * WM + l15) * kRowBytes, fb_row = (wn * WN + l15) * kRowBytes;
    // k-major right operand: a fragment is two transpose loads of 8 bytes.  The lanes work in groups of 16: lane t of a
    // group points at the 8 bytes that hold columns 4 (t % 4) .. + 3 of k row t / 4 (of the group's 4 k rows), and
    // receives column t of those 4 k rows.  Group g takes the block's 16 columns at k 8 g .. + 3 (second load: + 4 .. + 7).
    int fb_km[NI];
    if constexpr (BKM) {
        const int f = ((l15 >> 2) << 1) ^ ((g & 1) << 3);  // the unit swizzle of this lane's k rows
#pragma unroll
        for (int j = 0; j < NI; ++j)
            fb_km[j] = (8 * g + (l15 >> 2)) * (BN * 2) + (((wn * WN + j * 16) / 8 + ((l15 & 3) >> 1)) ^ f) * 16 + (l15 & 1) * 8;
    }
    int fa_km[MI];  // the same for a k-major left operand
    if constexpr (AKM) {
        const int f = ((l15 >> 2) << 1) ^ ((g & 1) << 3);
#pragma unroll
        for (int i = 0; i < MI; ++i)
            fa_km[i] = (8 * g + (l15 >> 2)) * (BM * 2) + (((wm * WM + i * 16) / 8 + ((l15 & 3) >> 1)) ^ f) * 16 + (l15 & 1) * 8;
    }
    // (absolute LDS addresses of the stage that is read next, changed over once a step)
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>(smem));
    uint32_t at_a[MI], at_b[NI];
    if constexpr (AKM)
#pragma unroll
        for (int i = 0; i < MI; ++i) at_a[i] = lds0 + fa_km[i];
    if constexpr (BKM)
#pragma unroll
        for (int j = 0; j < NI; ++j) at_b[j] = lds0 + kDenseA + fb_km[j];
    auto other_stage = [&] {
        static_assert(kDenseStage == 65536, "one address bit tells the stages apart");
        if constexpr (AKM)
#pragma unroll
            for (int i = 0; i < MI; ++i) at_a[i] ^= kDenseStage;
        if constexpr (BKM)
#pragma unroll
            for (int j = 0; j < NI; ++j) at_b[j] ^= kDenseStage;
    };
    auto read_tr = [&](uint32_t base, int ks) -> u32x4 {
        static_assert(BM == BN, "k rows of both operands have one length");
        const uint32_t at = base + uint32_t(ks * 32 * (BN * 2));
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at + 4 * (BN * 2)));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(u32x4, both);
    };
    auto read_a = [&](const char* sa, int i, int ks) -> u32x4 {
        if constexpr (AKM)
            return read_tr(at_a[i], ks);
        else
            return *reinterpret_cast<const u32x4*>(sa + fa_row + i * 16 * kRowBytes + koff[ks]);
    };
    auto read_b = [&](const char* sb, int j, int ks) -> u32x4 {
        if constexpr (BKM)
            return read_tr(at_b[j], ks);
        else
            return *reinterpret_cast<const u32x4*>(sb + fb_row + j * 16 * kRowBytes + koff[ks]);
    };

    const int nk = K / BK;
    u32x4 lw[4];  // the left operand's stage kt + 2 at the start of step kt
    loader.prologue(K);
    if constexpr (AKM) {
        left.prologue(nk, lw);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    } else {
        loader.first_stage_landed(nk);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Software pipeline over slices of 32 k, two per step.  A slice runs over the wave's blocks twice, first with the
    // column blocks 0, 1, then with 2, 3.  Every fragment register is loaded again, for the next slice, right behind its
    // last use: a row fragment in the second half, a pair of column fragments at the end of its half -- 14 to 16 MFMAs
    // before the next use, with one set of fragment registers (48; a second set would not fit beside the epilogues).
    // The compiler's own scheduler sinks every ds_read next to its first use (one exposed LDS latency per MFMA pair), so
    // the issue order is pinned explicitly: MFMA, then at most two fragment reads and one tile transfer.
    //
    // The barrier that frees a stage sits inside the step's second slice, kBarAt row blocks into its first half: by then
    // the last fragments of the stage, read at the end of the first slice, have arrived.  The stage's refill follows
    // it, one transfer every other MFMA, and has until the same place of the next step to land.
    //
    // Bound by power (clock 1.5-1.7 GHz) and the arrival of the tiles.  Forward and backward, of which the two products are
    // two thirds, against products on 32x32x16 MFMAs with two sets of fragments and the tile order of that time: 9664
    // tokens, H = 3584, V = 151936 27.7 -> 26.4 ms; 1396 tokens, H = 2048, V = 50257 1115 -> 1020 us; 459 tokens, H = 3584,
    // V = 151936 2554 -> 2300 us.
    constexpr int kBarAt = 4;
    static_assert(NI == 4 && 2 * kStageLoads <= 2 * (MI - kBarAt) + 2 * MI, "the refill fits behind the barrier");
    u32x4 a[MI], b[NI];
    {
        const char* sa = smem;
        const char* sb = smem + kDenseA;
        b[0] = read_b(sb, 0, 0);
        b[1] = read_b(sb, 1, 0);
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = read_a(sa, i, 0);
        b[2] = read_b(sb, 2, 0);
        b[3] = read_b(sb, 3, 0);
    }
    auto step = [&](int kt, auto refill_tag, auto next_tag) {
        constexpr bool REFILL = decltype(refill_tag)::value, NEXT = decltype(next_tag)::value;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            // the next slice: this stage's second, or the next stage's first
            const char* na = smem + ((kt + ks) & 1) * kDenseStage;
            const char* nb = na + kDenseA;
            const bool load = ks == 0 || NEXT;
            int issued = 0, slot = 0;
            if (ks == 1) other_stage();
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    if (ks == 1 && half == 0 && i == kBarAt) {
                        // Every fragment read of this stage has returned and the next stage has landed.  A bare s_barrier:
                        // __syncthreads() carries release / acquire fences; nothing may move across it.
                        // (with a left operand in registers the wait is one that the compiler counts: it need not wait for them again)
                        if constexpr (AKM)
                            __builtin_amdgcn_s_waitcnt(0);
                        else
                            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                        asm volatile("" ::: "memory");
                        __builtin_amdgcn_sched_barrier(0);
                        __builtin_amdgcn_s_barrier();
                        __builtin_amdgcn_sched_barrier(0);
                        asm volatile("" ::: "memory");
                    }
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        const int j = half * 2 + jj;
                        if constexpr (TURNED)
                            acc[i][j] = mfma<DT>(b[j], a[i], acc[i][j]);
                        else
                            acc[i][j] = mfma<DT>(a[i], b[j], acc[i][j]);
                        __builtin_amdgcn_sched_barrier(0);  // (a load moved above the MFMA would need registers of its own)
                        if (load) {
                            if (half == 1 && jj == 1) a[i] = read_a(na, i, ks ^ 1);
                            if (i == MI - 1) b[j] = read_b(nb, j, ks ^ 1);
                        }
                        if (REFILL && ks == 1 && (half == 1 || i >= kBarAt)) {
                            if ((AKM ? slot % 3 == 2 : (slot & 1)) && issued < kStageLoads) {
                                loader.issue_one(kt & 1, (kt + 2) * BK, issued);
                                ++issued;
                            }
                            // a pair of columns behind two of three MFMAs (its six instructions keep the vector unit as busy as
                            // three MFMAs of the SIMD's two waves do the matrix unit); a vector that is whole makes room
                            // for the next stage's
                            if constexpr (AKM) {
                                if (slot % 3 != 2) {
                                    const int pair = slot - slot / 3;
                                    uint32_t x = lw[pair >> 2][pair & 3];
                                    left.convert(x);
                                    lw[pair >> 2][pair & 3] = x;
                                    if ((pair & 3) == 3) {
                                        left.store(kt & 1, pair >> 2, lw[pair >> 2]);
                                        left.load(min(kt + 3, nk - 1) * BK, pair >> 2, lw[pair >> 2]);
                                    }
                                }
                            }
                            ++slot;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };
    constexpr std::true_type T{};
    constexpr std::false_type F{};
    int kt = 0;
    for (; kt + 2 < nk; ++kt) step(kt, T, T);
    if (kt + 1 < nk) step(kt++, F, T);
    step(kt, F, F);
    // every LDS read of this tile completed before the last barrier: the caller may reuse the LDS right away
}

// Row (M index) inside the workgroup tile of accumulator element r of block i, for this lane.
__device__ __forceinline__ int acc_row(int wm, int i, int r, int lane) { return wm * WM + i * 16 + (lane >> 4) * 4 + r; }
// Column (N index) inside the workgroup tile of block j, for this lane.
__device__ __forceinline__ int acc_col(int wn, int j, int lane) { return wn * WN + j * 16 + (lane & 15); }
// The same with TURNED: the row of block i, and the column of element 0 of block j.
__device__ __forceinline__ int acc_turned_row(int wm, int i, int lane) { return wm * WM + i * 16 + (lane & 15); }
__device__ __forceinline__ int acc_turned_col(int wn, int j, int lane) { return wn * WN + j * 16 + (lane >> 4) * 4; }

// Workgroup id -> (tile along axis `a`, tile along axis `b`) such that the workgroups that run
// together on one XCD (ids congruent mod 8, dispatched round-robin) form patches of about 4 x 8 tiles: they share
// operand slabs through that XCD's L2.  No workgroup of the grid but a few at the end is empty: the hardware deals
// workgroups to the CUs in order, and with empty ones interleaved at a fixed stride the real ones end up on a fraction of
// the CUs (measured: a third more time for 65 instead of 64 a tiles with a grid padded to whole bands).
//
// From 32 a tiles on an XCD owns the `a` tiles congruent to its number mod 8, in bands of 4; inside a band it walks b
// with the band's a tiles innermost.  The last band holds only as many a tiles per XCD as n_a needs.  The n_a % 8 a tiles
// that are left when every XCD has the same number are not given to that many XCDs whole (one XCD in eight would then
// carry an a tile more than the others and the launch would wait for it): their n_b tiles each are dealt out
// in equal runs over all eight XCDs, a innermost.
//
// Fewer a tiles (token counts below 8192) are put into even bands of at most 8; inside a band b is walked with the band's a
// tiles innermost, and each XCD takes one eighth of that sequence: 4 to 8 a tiles beside 4 to 8 b tiles at a time.  Under
// the rule for many a tiles an XCD has ONE a tile beside 32 b tiles when there are 8 to 15, and fetches 33 slabs where
// 12 would do: 2300 tokens, H = 2048, V = 128256 forward 1140 -> 1107 us, with backward 3720 -> 3690 us; 1000 tokens,
// H = 2048, V = 128256 (there the slices of dHidden) 1948 -> 1918 us.
// The same for the last few of many a tiles loses (79 a tiles: forward 3653 -> 3735 us).
// The caller skips ta >= n_a or tb >= n_b.
__device__ __forceinline__ void xcd_patch(int w, int n_a, int n_b, int& ta, int& tb) {
    const int xcd = w & 7, q = w >> 3;
    const int groups = n_a >= 32 ? n_a >> 3 : 0;   // a tiles every XCD owns whole
    const int bands = groups >> 2;                 // full bands of 4 of them
    const int full = bands * 4 * n_b;              // workgroups of this XCD in the full bands
    const int m = groups & 3;                      // whole a tiles per XCD in the last band
    if (q < full) {
        const int rem = q % (4 * n_b);
        tb = rem >> 2;
        ta = ((q / (4 * n_b)) * 4 + (rem & 3)) * 8 + xcd;
        return;
    }
    if (q < full + m * n_b) {
        const int qq = q - full;
        tb = qq / m;
        ta = (bands * 4 + qq % m) * 8 + xcd;
        return;
    }
    // the a tiles that are left, from n_a - left on, dealt out in runs
    const int left = n_a - groups * 8, share = (left * n_b + 7) >> 3, i = q - full - m * n_b, t = xcd * share + i;
    if (i >= share || t >= left * n_b) {
        ta = n_a;
        tb = n_b;
        return;
    }
    const int n_bands = (left + 7) >> 3, narrow = left / n_bands, wide = left % n_bands;  // `wide` bands of narrow + 1, then narrow
    const int in_wide = wide * (narrow + 1) * n_b;
    const int width = t < in_wide ? narrow + 1 : narrow, u = t < in_wide ? t : t - in_wide;
    const int band = u / (width * n_b), v = u - band * (width * n_b);
    tb = v / width;
    ta = groups * 8 + (t < in_wide ? 0 : wide * (narrow + 1)) + band * width + (v - tb * width);
}
inline int xcd_patch_grid(int n_a, int n_b) {
    const int groups = n_a >= 32 ? n_a / 8 : 0, left = n_a - groups * 8;
    return 8 * (groups * n_b + (left * n_b + 7) / 8);
}

}  // namespace
}  // namespace trlk
