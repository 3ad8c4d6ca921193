// Products of 8-bit floating-point operands with an fp32 scale for each block of 128 along K:
//
//   c[m, n] = sum_kb sa[m, kb] * sb[n / 128 or n, kb] * sum_{k in block kb} a[m, k] * b[n, k]
//
// dense, or for ragged groups of rows that each have a b of their own.  One v_mfma_f32_16x16x128_f8f6f4 is a whole block of K, so it starts from zero
// and its four sums a lane go into fp32 accumulators by four multiply-adds with sa * sb (a product rounded to fp32; with a scale for each row of b by
// sb first).  A scale that is no power of two cannot go through the matrix instruction, and the vector unit reaches no AGPR: the accumulators lie in
// VGPRs and the multiply-adds, half the matrix pipe's time, run beside it.  Which K of a block a lane holds is the same for both operands, so a lane takes its
// 16-byte pieces as memory has them.
//
// Two kernels: fp8_rows_kernel for few rows (K shared out over the wavefronts of a workgroup, operands straight into registers), fp8_tile_kernel else
// (tiles through the LDS).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mx_gemm_common.h"
#include "mx_launch.h"

namespace cmx {
namespace {

constexpr uint32_t kBlockK = 128;

struct Fp8GemmArgs {
    const uint8_t *a, *b;
    const float *a_scale, *b_scale;
    uint8_t* c;
    const int32_t* sizes;                 // [groups] or null
    size_t b_step, bs_step;               // from group to group: bytes, elements
    uint32_t lda, ldb, ld_as, ld_bs, ldc;
    uint32_t m, n, k, blocks, groups, n_tiles, zero_rest;
    int out_type;
    float* parts;                         // sums of the blocks of K that each of `splits` workgroups to a tile has, [splits][m][n_wide], or null
    uint32_t split_blocks, n_wide;
};

// What a workgroup computes: `rows` rows from row0 on of group g, or (g == groups) zeros into rows behind the groups
struct Work {
    uint32_t g, row0, rows, n_tile;
};

// Work item `id` of a launch whose tiles have TM rows: m-tiles of a group run fastest, so that neighbours share its weights.  Every wavefront scans the group
// sizes, four to a lane.  Negative sizes count as zero, rows past m do not exist.
template <uint32_t TM>
__device__ __forceinline__ bool locate(const Fp8GemmArgs& p, uint32_t id, Work& w, bool xcd_runs) {
    if (p.sizes == nullptr) {
        const uint32_t m_tiles = (p.m + TM - 1) / TM, total = m_tiles * p.n_tiles;
        if (id >= total) return false;
        const uint32_t l = xcd_runs ? tile_of_workgroup(total, id) : id;
        constexpr uint32_t kBand = 8;
        const uint32_t band = l / (kBand * p.n_tiles), in = l % (kBand * p.n_tiles), high = min(kBand, m_tiles - band * kBand);
        w.g = 0;
        w.row0 = (band * kBand + in % high) * TM;
        w.rows = min(TM, p.m - w.row0);
        w.n_tile = in / high;
        return true;
    }
    const uint32_t lane = threadIdx.x & 63u, m = p.m;
    const auto add = [](uint32_t x, uint32_t y) -> uint32_t { return x + y; };
    const auto sat = [m](uint32_t x, uint32_t y) -> uint32_t { return min(x + y, m); };          // x, y <= m < 2^31
    // tiles of all groups first: the order of the workgroups hangs on their number
    uint32_t all_tiles = 0, all_rows = 0;
    uint32_t rows[4], first = 0, tile_end = 0, row_end = 0;
    for (uint32_t pass = 0, at = 0, l = 0; pass < 2; ++pass) {
        uint32_t tiles_before = 0, rows_before = 0;
        for (uint32_t g0 = 0; g0 < p.groups; g0 += 256) {
            if (pass == 0 || p.groups > 256) {
                uint32_t sum = 0;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t g = g0 + 4 * lane + j;
                    const int32_t v = g < p.groups ? p.sizes[g] : 0;
                    rows[j] = v > 0 ? min((uint32_t)v, m) : 0u;
                    sum = sat(sum, rows[j]);
                }
                row_end = sat(wave_scan(sum, sat), rows_before);
                const uint32_t shifted = (uint32_t)__shfl_up((int)row_end, 1);
                first = lane == 0 ? rows_before : shifted;
                uint32_t from = first, tiles = 0;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t to = sat(from, rows[j]);
                    rows[j] = to - from;
                    tiles += (rows[j] + TM - 1) / TM;
                    from = to;
                }
                tile_end = wave_scan(tiles, add);
            }
            const uint32_t tiles_here = (uint32_t)__builtin_amdgcn_readlane((int)tile_end, 63);
            if (pass == 1) {
                const uint64_t found = __ballot((uint64_t)(tiles_before + tile_end) * p.n_tiles > l);
                if (found != 0) {
                    at = (uint32_t)__builtin_ctzll(found);
                    const uint32_t own = (rows[0] + TM - 1) / TM + (rows[1] + TM - 1) / TM + (rows[2] + TM - 1) / TM + (rows[3] + TM - 1) / TM;
                    uint32_t t0 = tiles_before + (uint32_t)__builtin_amdgcn_readlane((int)(tile_end - own), (int)at);
                    uint32_t r0 = (uint32_t)__builtin_amdgcn_readlane((int)first, (int)at);
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)rows[j], (int)at), t = (r + TM - 1) / TM;
                        if (l >= t0 * p.n_tiles && l < (t0 + t) * p.n_tiles) {
                            constexpr uint32_t kBand = 8;
                            const uint32_t in_group = l - t0 * p.n_tiles, band = in_group / (kBand * p.n_tiles), in = in_group % (kBand * p.n_tiles);
                            const uint32_t high = min(kBand, t - band * kBand);
                            w.g = g0 + 4 * at + j;
                            w.row0 = r0 + (band * kBand + in % high) * TM;
                            w.rows = min(TM, r0 + r - w.row0);
                            w.n_tile = in / high;
                        }
                        t0 += t;
                        r0 += r;
                    }
                    return true;
                }
            }
            tiles_before += tiles_here;
            rows_before = (uint32_t)__builtin_amdgcn_readlane((int)row_end, 63);
        }
        if (pass == 0) {
            all_tiles = tiles_before;
            all_rows = rows_before;
            const uint32_t total = all_tiles * p.n_tiles;
            if (id >= total) {
                if (!p.zero_rest) return false;
                const uint32_t behind = id - total;
                w.g = p.groups;
                w.n_tile = behind % p.n_tiles;
                w.row0 = all_rows + behind / p.n_tiles * TM;
                if (w.row0 >= m || w.row0 < all_rows) return false;
                w.rows = min(TM, m - w.row0);
                return true;
            }
            l = xcd_runs ? tile_of_workgroup(total, id) : id;
        }
    }
    return false;
}

// four consecutive results, or as many as `left`, to column n of a row
__device__ __forceinline__ void store4(uint8_t* row, uint32_t n, const v4f v, int type, uint32_t left) {
    uint32_t w[4];
    if (type == CMX_OUT_FP32) {
        float* const p = reinterpret_cast<float*>(row) + n;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
        if (left >= 4) __builtin_memcpy(p, w, 16);
        else
            for (uint32_t i = 0; i < left; ++i) p[i] = v[i];
        return;
    }
    if (type == CMX_OUT_BF16) {
        w[0] = cvt_pk_bf16(v[0], v[1]);
        w[1] = cvt_pk_bf16(v[2], v[3]);
    } else {
        typedef _Float16 v2f16 __attribute__((ext_vector_type(2)));
        w[0] = __builtin_bit_cast(uint32_t, (v2f16){(_Float16)v[0], (_Float16)v[1]});
        w[1] = __builtin_bit_cast(uint32_t, (v2f16){(_Float16)v[2], (_Float16)v[3]});
    }
    uint16_t* const p = reinterpret_cast<uint16_t*>(row) + n;
    if (left >= 4) {
        __builtin_memcpy(p, w, 8);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
        if (i < left) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
}

__device__ __forceinline__ void zero_tile(const Fp8GemmArgs& p, const Work& w, uint32_t n0, uint32_t tn) {
    const uint32_t size = p.out_type == CMX_OUT_FP32 ? 4 : 2, quads = tn / 4;
    for (uint32_t i = threadIdx.x; i < w.rows * quads; i += blockDim.x) {
        const uint32_t n = n0 + 4 * (i % quads);
        if (n < p.n) store4(p.c + (size_t)(w.row0 + i / quads) * p.ldc * size, n, (v4f){0, 0, 0, 0}, p.out_type, p.n - n);
    }
}

template <int FMT>
__device__ __forceinline__ v4f block_product(const v8i& b, const v8i& a) {
    constexpr int kF = FMT == CMX_FMT_E5M2 ? 1 : 0;
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, (v4f){0, 0, 0, 0}, kF, kF, 0, 0, 0, 0);
}

template <int I, int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

// Rows of 128 bytes in LDS: row r holds its 16-byte piece p at place p ^ (r / 2 % 8), so that the 16 rows that a fragment reads at a time lie in different banks
__device__ __forceinline__ uint32_t place_of(uint32_t row, uint32_t piece) { return piece ^ ((row >> 1) & 7u); }

// Between LDS writes of some lanes and reads of the same wavefront's others, or the other way round: the LDS takes a wavefront's accesses in order, so only the compiler, which
// sees one lane, has to keep them so.  No instruction
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// ---- few rows ------------------------------------------------------------------------------------------------------------
// A workgroup owns 16 FN columns of c and 16 FM rows over all of K; its wavefronts take the blocks of K in turn, DEPTH of each in flight, and join their
// sums in LDS in the order of the wavefronts.  Loads take whole lines (8 rows of 128 bytes); lane l of a fragment holds row l % 16, the 16-byte pieces l / 16 and l / 16 + 4
// of a block, so operands change lanes through the LDS (loads as fragments want them, 16 rows of 64 bytes, cost the vector cache twice as much: 16 rows of 4096 x 7168
// 10.7 us, so 8.2; 64 rows 18.3, so 12.6).
// Bound by reading the weights where rows are few: one row of 4096 x 7168 in 7.3 us (4.0 TB/s, 2.5 of it the launch), 256 rows on 256 experts of 7168 x 2048 in 400 us (5.9 TB/s);
// by loads of operands where they are more: 64 rows of 4096 x 7168 pull 458 KB into each CU in 12.9 us, of which loads alone take 11.9 (half of them weights that two XCDs fetch each for
// itself: the row tiles of the same columns are neighbours in number).  Deeper rings change nothing (64 rows: 2 blocks 12.6, 3 13.1, 4 13.6).
template <int FMT, int FN, int FM, int DEPTH, bool ROW_SCALES>
__global__ __launch_bounds__(FN * FM == 1 ? 1024 : 512) void fp8_rows_kernel(const Fp8GemmArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr uint32_t TN = 16 * FN, TM = 16 * FM;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t r16 = lane & 15u, quarter = lane >> 4;
    Work w;
    if (!locate<TM>(p, blockIdx.x, w, false)) return;
    const uint32_t n0 = w.n_tile * TN;
    if (w.g == p.groups && p.sizes != nullptr) {
        zero_tile(p, w, n0, TN);
        return;
    }
    // a lane's rows of a fragment's two loads (8 rows of 128 bytes each), and the scales of the row or rows that its sums belong to
    const uint32_t row8 = lane >> 3, piece = lane & 7u;
    const uint8_t* const b0 = p.b + w.g * p.b_step + (size_t)n0 * p.ldb;
    const uint8_t* const a0 = p.a + (size_t)w.row0 * p.lda;
    uint32_t b_off[FN][2], a_off[FM][2];
    const float *b_scale[FN], *a_scale[FM];
    const uint32_t n_left = p.n - n0;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) b_off[i][h] = min(16 * i + 8 * h + row8, n_left - 1) * p.ldb;
        b_scale[i] = p.b_scale + w.g * p.bs_step + (ROW_SCALES ? (size_t)min(n0 + 16 * i + 4 * quarter, p.n - 1) * p.ld_bs : (size_t)((n0 + 16 * i) / kBlockK) * p.ld_bs);
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) a_off[j][h] = min(16 * j + 8 * h + row8, w.rows - 1) * p.lda;
        a_scale[j] = p.a_scale + (size_t)(w.row0 + min(16 * j + r16, w.rows - 1)) * p.ld_as;
    }
    v4f sum[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) sum[i][j] = (v4f){0, 0, 0, 0};
    // the rows of b behind the lane's first that its four sums belong to
    uint32_t bs_at[FN][4];
    if constexpr (ROW_SCALES) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t n = n0 + 16 * i + 4 * quarter;
                bs_at[i][r] = n + r < p.n ? r : (n < p.n ? p.n - 1 - n : 0);
            }
    }
    // pieces behind K repeat the last one of the row, and are cleared before they count
    const uint32_t last = p.blocks - 1, far = p.k - 16, tail = p.k % kBlockK;
    uint8_t* const stage = smem + wave * ((FN + FM) * 16 * kBlockK);
    const uint32_t put = row8 * kBlockK, get = r16 * kBlockK + 16 * place_of(r16, quarter);
    // the fragment of 16 rows out of what their two loads brought, through a piece of LDS that is this wavefront's alone
    const auto exchanged = [&](v4i (&v)[2], int slot, bool clear) -> v8i {
        uint8_t* const at = stage + slot * (16 * kBlockK);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            if (clear) v[h] = (v4i){0, 0, 0, 0};
            *reinterpret_cast<v4i*>(at + put + h * (8 * kBlockK) + 16 * place_of(8 * h + row8, piece)) = v[h];
        }
        wave_fence();
        const v4i lo = *reinterpret_cast<const v4i*>(at + get), hi = *reinterpret_cast<const v4i*>(at + (get ^ 64u));
        wave_fence();
        return (v8i){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    v4i b[DEPTH][FN][2], a[DEPTH][FM][2];
    float sb[DEPTH][FN][ROW_SCALES ? 4 : 1], sa[DEPTH][FM];
    const auto load = [&](auto d_c, uint32_t kb) {
        constexpr int d = decltype(d_c)::value;
        const uint32_t at = min(kb * kBlockK + 16 * piece, far);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) b[d][i][h] = *reinterpret_cast<const v4i*>(b0 + (b_off[i][h] + at));
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) a[d][j][h] = *reinterpret_cast<const v4i*>(a0 + (a_off[j][h] + at));
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            if constexpr (ROW_SCALES) {
#pragma unroll
                for (int r = 0; r < 4; ++r) sb[d][i][r] = b_scale[i][(size_t)bs_at[i][r] * p.ld_bs + kb];
            } else {
                sb[d][i][0] = b_scale[i][kb];
            }
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) sa[d][j] = a_scale[j][kb];
    };
    const auto multiply = [&](auto d_c, uint32_t kb) {
        constexpr int d = decltype(d_c)::value;
        const bool clear = tail != 0 && kb == last && 16 * piece >= tail;
        v8i af[FM];
#pragma unroll
        for (int j = 0; j < FM; ++j) af[j] = exchanged(a[d][j], FN + j, clear);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const v8i bf = exchanged(b[d][i], i, clear);
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const v4f part = block_product<FMT>(bf, af[j]);
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[i][j][r] = __builtin_fmaf(part[r], sa[d][j] * sb[d][i][ROW_SCALES ? r : 0], sum[i][j][r]);
            }
            if constexpr (FN * FM >= 8) __builtin_amdgcn_sched_barrier(0);      // (one fragment of b at a time: registers)
        }
    };
    // (workgroups have no more wavefronts than there are blocks)
    static_for<0, DEPTH>([&](auto d) {
        if (wave + d * waves < p.blocks) load(d, wave + d * waves);
    });
    for (uint32_t kb0 = wave; kb0 < p.blocks; kb0 += DEPTH * waves)
        static_for<0, DEPTH>([&](auto d) {
            const uint32_t kb = kb0 + d * waves;
            if (kb >= p.blocks) return;
            multiply(d, kb);
            if (kb + DEPTH * waves < p.blocks) load(d, kb + DEPTH * waves);
        });
    __syncthreads();
    v4f* const sums = reinterpret_cast<v4f*>(smem);
    constexpr uint32_t kEach = FN * FM * 64;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) sums[wave * kEach + (i * FM + j) * 64 + lane] = sum[i][j];
    __syncthreads();
    const uint32_t size = p.out_type == CMX_OUT_FP32 ? 4 : 2;
    for (uint32_t at = threadIdx.x; at < kEach; at += blockDim.x) {
        v4f v = sums[at];
        for (uint32_t u = 1; u < waves; ++u) v += sums[u * kEach + at];
        const uint32_t l = at & 63u, t = at >> 6, row = t % FM * 16 + (l & 15u), n = n0 + t / FM * 16 + 4 * (l >> 4);
        if (row < w.rows && n < p.n) store4(p.c + (size_t)(w.row0 + row) * p.ldc * size, n, v, p.out_type, p.n - n);
    }
}

// ---- tiles through the LDS -------------------------------------------------------------------------------------------------
// A workgroup of WN x WM wavefronts owns TN columns and TM rows of c.  Blocks of K travel by LDS-DMA into SLOTS slots.
// Two wavefronts to a SIMD share the matrix pipe and the vector unit: products and multiply-adds alone, without memory, run at 3.84 PFLOP/s (32 x 32 x 64 products: 3.36).  A
// wavefront's 128 x 64 of c are 128 accumulators; 128 x 128 would not leave the vector unit a register.  256 x 256 tiles, 8192 x 4096 x 7168: 216 - 224 us (2.2 PFLOP/s), the matrix
// pipe busy for 47 - 53 % of a clock that the chip lowers to 1.8 - 2.2 GHz under it.  Of 231 us in one run of it, without the multiply-adds 199, without the loads of operands 172,
// without both 156.  With a scale for each row of b twice the vector work: 4096 x 2048 x 2784 37 us (31 with one for 128 rows), a block of K 1.37: 0.27 of it waits for loads, 0.43 are
// multiply-adds (0.24 the products of scales), 0.66 products, barriers and LDS reads; they add up, and no unit is full (matrix pipe 23 %, vector unit 30 %).
__device__ __forceinline__ uint32_t same(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ void dma16(uint32_t lds, uint32_t off, v4i rsrc, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(same(lds)), "v"(off), "s"(rsrc), "s"(same(soff)) : "memory");
}
__device__ __forceinline__ v4i buffer_at(const uint8_t* base) {
    const uint64_t v = reinterpret_cast<uint64_t>(base);
    return (v4i){(int)same((uint32_t)v), (int)same((uint32_t)(v >> 32)), (int)0x80000000u, 0x00020000};      // offsets of 2^31 on give zeros
}

// blocks of K whose scales lie in LDS at a time (twice)
template <bool ROW_SCALES>
constexpr uint32_t kSpanOf = ROW_SCALES ? 4 : 8;

template <int FMT, int TN, int TM, int WN, int WM, int SLOTS, bool ROW_SCALES>
__global__ __launch_bounds__(64 * WN * WM) void fp8_tile_kernel(const Fp8GemmArgs args) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr uint32_t NW = WN * WM, NT = 64 * NW, FN = TN / WN / 16, FM = TM / WM / 16, kRows = TN + TM, kSlot = kRows * kBlockK;
    constexpr uint32_t kLoads = kRows / (8 * NW), kBLoads = TN / (8 * NW);
    constexpr uint32_t kScaleSpan = kSpanOf<ROW_SCALES>, kScaleRows = TM + (ROW_SCALES ? TN : 0), kScaleBase = SLOTS * kSlot, kScaleHalf = kScaleRows * kScaleSpan * 4;
    static_assert(TN % (8 * NW) == 0 && TM % (8 * NW) == 0 && (8 * NW) % 16 == 0, "loads of whole rows, the same piece in all of a lane's");
    static_assert(128 % (TN / WN) == 0, "a wavefront's columns share a scale");
    // loads of a block behind the last products of the block before its slot's last one, and products that the others are spread over
    constexpr uint32_t kEarly = FM < kLoads / 2 ? FM : kLoads / 2, kLate = kLoads - kEarly, kSpread = std::max(kLate, FN * FM / 4);
    static_assert(FM >= 3 && FN % 2 == 0 && kSpread <= (FN - 1) * FM, "fragments and scales change places behind their last use; loads stand in front of the wait");
    Fp8GemmArgs p = args;
    if (p.parts != nullptr) {                                          // this workgroup's blocks of K as a problem of their own
        const uint32_t from = blockIdx.y * p.split_blocks;
        p.blocks = min(p.split_blocks, p.blocks - from);
        p.a += from * kBlockK;
        p.b += from * kBlockK;
        p.a_scale += from;
        p.b_scale += from;
        p.k = min(p.blocks * kBlockK, p.k - from * kBlockK);
    }
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = same(tid >> 6), wn = wave % WN, wm = wave / WN, r16 = lane & 15u, quarter = lane >> 4;
    Work w;
    if (!locate<TM>(p, blockIdx.x, w, true)) return;
    w.g = same(w.g); w.row0 = same(w.row0); w.rows = same(w.rows); w.n_tile = same(w.n_tile);
    const uint32_t n0 = w.n_tile * TN;
    if (w.g == p.groups && p.sizes != nullptr) {
        zero_tile(p, w, n0, TN);
        return;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    const v4i b_buf = buffer_at(p.b + w.g * p.b_step + (size_t)n0 * p.ldb), a_buf = buffer_at(p.a + (size_t)w.row0 * p.lda);
    const uint32_t n_rows = min((uint32_t)TN, p.n - n0);

    // load i of this wavefront: rows (NW i + wave) * 8 .. + 8 of the slot, lane -> row lane / 8, place lane % 8; rows that do not exist repeat the last
    uint32_t off[kLoads];
    const uint32_t my_piece = place_of(wave * 8 + (lane >> 3), lane & 7u);
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t r = (NW * i + wave) * 8 + (lane >> 3);
        off[i] = (i < kBLoads ? min(r, n_rows - 1) * p.ldb : min(r - TN, w.rows - 1) * p.lda) + 16 * my_piece;
    }
    const uint32_t last = p.blocks - 1, behind = last * kBlockK + 16 * my_piece < p.k ? 0u : 0x80000000u;      // pieces behind K, in its last block
    // load i of block kb; past the last block zeros come without a look at memory, so that every block counts the same loads
    const auto gone = [&](uint32_t kb) -> uint32_t { return kb < last ? 0u : (kb == last ? behind : 0x80000000u); };
    const auto issue = [&](uint32_t kb, uint32_t slot, uint32_t i, uint32_t gone) {
        dma16(lds0 + slot * kSlot + (NW * i + wave) * 1024, off[i] | gone, i < kBLoads ? b_buf : a_buf, kb * kBlockK);
    };
    // Two slots: a block's loads have less than a block's time, so lines that are not in the L2 by then stop everybody.  Of the workgroups that work on the same rows
    // of an operand at the same time (8 x 4 tiles on an XCD, as locate numbers them) each asks for a share of the lines of a later block, a dword of each, into LDS
    // that nobody reads (16 experts of 32768 rows 955 -> 910 us in one run, all lines by every workgroup 1056; runs of the kernel as it is differ from 940 to 978; with three slots nothing is gained).
    constexpr bool kTouch = SLOTS == 2;
    constexpr uint32_t kAhead = 3;
    const uint32_t in_band = (w.row0 / TM) % 8, in_chunk = w.n_tile % 4;
    const uint32_t line_row = wave == 0 ? in_chunk * (TM / 4) + lane : in_band * (TN / 8) + (lane & (TN / 8 - 1));
    const uint32_t line_off = wave == 0 ? min(line_row, w.rows - 1) * p.lda : min(line_row, n_rows - 1) * p.ldb;
    const v4i line_buf = wave == 0 ? a_buf : b_buf;
    const auto touch = [&](uint32_t kb) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(same(lds0 + kScaleBase + 2 * kScaleHalf + wave * 256)),
                     "v"(kb <= last ? line_off : 0x80000000u), "s"(line_buf), "s"(same(kb * kBlockK)) : "memory");
    };
    // scales of blocks span * kScaleSpan .. + kScaleSpan, [block][row], into half span % 2; a thread has some rows' four blocks
    // (fetched in a span's first block; placed at the end of a block that has another one's barrier between it and the last, where they are read first)
    constexpr uint32_t kPlace = kScaleSpan - 3;
    constexpr uint32_t kPieces = kScaleRows * (kScaleSpan / 4), kMine = (kPieces + NT - 1) / NT;
    float staged[kMine][4];
    const auto fetch_scales = [&](uint32_t span) {
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint32_t at = min(tid + i * NT, kPieces - 1), row = at / (kScaleSpan / 4), kb = span * kScaleSpan + 4 * (at % (kScaleSpan / 4));
            const float* const s = row < TM ? p.a_scale + (size_t)(w.row0 + min(row, w.rows - 1)) * p.ld_as
                                            : p.b_scale + w.g * p.bs_step + (size_t)(n0 + min(row - TM, n_rows - 1)) * p.ld_bs;
            if (kb + 4 <= p.blocks) {
                __builtin_memcpy(staged[i], s + kb, 16);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) staged[i][j] = s[min(kb + j, last)];
            }
        }
    };
    const auto place_scales = [&](uint32_t span) {
        float* const half = reinterpret_cast<float*>(smem + kScaleBase + (span & 1u) * kScaleHalf);
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint32_t at = tid + i * NT;
            if (kPieces % NT == 0 || at < kPieces) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) half[(4 * (at % (kScaleSpan / 4)) + j) * kScaleRows + at / (kScaleSpan / 4)] = staged[i][j];
            }
        }
    };
    typedef const __attribute__((address_space(4))) float* scalar_f32;
    const scalar_f32 b_scale = (scalar_f32)(p.b_scale + w.g * p.bs_step + (size_t)min((n0 + wn * (TN / WN)) / kBlockK, (p.n - 1) / kBlockK) * p.ld_bs);

    v4f sum[FN][FM];
#pragma unroll
    for (uint32_t i = 0; i < FN; ++i)
#pragma unroll
        for (uint32_t j = 0; j < FM; ++j) sum[i][j] = (v4f){0, 0, 0, 0};
    // a fragment's rows are 16 apart from those of the next: their pieces lie at the same places, and the second 64 bytes at the first's with one bit turned
    const uint32_t in_rows = r16 * kBlockK + 16 * place_of(r16, quarter);
    const uint32_t b_lo = wn * (TN / WN) * kBlockK + in_rows, a_lo = (TN + wm * (TM / WM)) * kBlockK + in_rows;
    const auto fragment = [&](uint32_t lo, uint32_t i) -> v8i {
        typedef __attribute__((address_space(3))) const v4i* lds_v4i;
        const v4i x = *(lds_v4i)(uintptr_t)(lo + i * (16 * kBlockK)), y = *(lds_v4i)(uintptr_t)((lo ^ 64u) + i * (16 * kBlockK));
        return (v8i){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };

#pragma unroll
    for (uint32_t d = 0; d + 1 < SLOTS; ++d)
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) issue(d, d, i, gone(d));
#pragma unroll
    for (uint32_t i = 0; i < kEarly; ++i) issue(SLOTS - 1, SLOTS - 1, i, gone(SLOTS - 1));
    fetch_scales(0);
    place_scales(0);
    v8i a[FM], b[2];
    float s[FM], s_next[FM];
    v4f part[4], rs[2];
    const uint32_t b_row = wn * (TN / WN), a_row = wm * (TM / WM) + r16;
    const auto scales_of = [&](uint32_t kb) -> const float* {
        return reinterpret_cast<const float*>(smem + kScaleBase + (kb / kScaleSpan & 1u) * kScaleHalf) + kb % kScaleSpan * kScaleRows;
    };
    const auto row_scales = [&](const float* scales, uint32_t i) { rs[i & 1] = *reinterpret_cast<const v4f*>(scales + TM + b_row + 16 * i + 4 * quarter); };
    const auto add = [&](uint32_t x) {
        const uint32_t i = x / FM, j = x % FM;
        asm volatile("" : "+v"(part[x % 4]));                          // (not in AGPRs, from which the vector unit would have to copy it)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if constexpr (ROW_SCALES) sum[i][j][r] = __builtin_fmaf(part[x % 4][r], rs[i & 1][r] * s[j], sum[i][j][r]);
            else sum[i][j][r] = __builtin_fmaf(part[x % 4][r], s[j], sum[i][j][r]);
        }
        asm volatile("" : "+v"(sum[i][j]));                            // (used here: the compiler would put all multiply-adds behind all products)
    };
    float sb = ROW_SCALES ? 0.0f : b_scale[0];
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((SLOTS - 2) * kLoads + kEarly) : "memory");
    // A wavefront whose rows do not exist (a group's last tile is half empty on average) only brings its share of the operands
    if (wm * (TM / WM) >= w.rows) {
        uint32_t slot = 0;
        for (uint32_t kb = 0; kb < p.blocks; ++kb) {
            const uint32_t span = kb / kScaleSpan, in_span = kb % kScaleSpan, before = slot == 0 ? SLOTS - 1 : slot - 1;
            const bool more = (span + 1) * kScaleSpan < p.blocks;
            if (in_span == 0 && more) fetch_scales(span + 1);
            if constexpr (kTouch)
                if (wave < 2) touch(kb + kAhead);
#pragma unroll
            for (uint32_t l = kEarly; l < kLoads; ++l) issue(kb + SLOTS - 1, before, l, gone(kb + SLOTS - 1));
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((SLOTS - 2) * kLoads) : "memory");
#pragma unroll
            for (uint32_t l = 0; l < kEarly; ++l) issue(kb + SLOTS, slot, l, gone(kb + SLOTS));
            if (in_span == kPlace && more) place_scales(span + 1);
            slot = slot + 1 < SLOTS ? slot + 1 : 0;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        return;
    }
    b[0] = fragment(lds0 + b_lo, 0);
    if constexpr (ROW_SCALES) row_scales(scales_of(0), 0);
#pragma unroll
    for (uint32_t j = 0; j < FM; ++j) {
        a[j] = fragment(lds0 + a_lo, j);
        s[j] = scales_of(0)[a_row + 16 * j];
        if constexpr (!ROW_SCALES) s[j] *= sb;
    }
    uint32_t slot = 0;
    for (uint32_t kb = 0; kb < p.blocks; ++kb) {
        const uint32_t span = kb / kScaleSpan, in_span = kb % kScaleSpan, before = slot == 0 ? SLOTS - 1 : slot - 1, next = slot + 1 < SLOTS ? slot + 1 : 0;
        const uint32_t gone_before = gone(kb + SLOTS - 1), gone_here = gone(kb + SLOTS), at = lds0 + slot * kSlot, next_at = lds0 + next * kSlot;
        const bool more = (span + 1) * kScaleSpan < p.blocks;
        if (in_span == 0 && more) fetch_scales(span + 1);
        const float *const scales = scales_of(kb), *const next_scales = scales_of(kb + 1);
        if constexpr (!ROW_SCALES) sb = b_scale[min(kb + 1, last)];
        if constexpr (kTouch)
            if (wave < 2) touch(kb + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        // A product, the multiply-adds of the one three before, its share of the loads: in this order.  In front of the last FM products every fragment of the block
        // has been read and the next block has arrived, for all: behind them go the reads of its first fragments and the first loads into the slot that is free now.
#pragma unroll
        for (uint32_t x = 0; x < FN * FM; ++x) {
            const uint32_t i = x / FM, j = x % FM;
            if (x == (FN - 1) * FM) {
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((SLOTS - 2) * kLoads) : "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
            part[x % 4] = block_product<FMT>(b[i & 1], a[j]);
            if constexpr (FN >= 4) __builtin_amdgcn_sched_barrier(0);        // (reads in front of a product would be waited for with its own)
            if (x >= 3) add(x - 3);
            if (x == FM + 2) {
#pragma unroll
                for (uint32_t l = 0; l < FM; ++l) s_next[l] = next_scales[a_row + 16 * l];
            }
            if (i + 1 < FN) {
                if (j == 0) b[(i + 1) & 1] = fragment(at + b_lo, i + 1);
                if constexpr (ROW_SCALES)
                    if (j == FM - 1) row_scales(scales, i + 1);
#pragma unroll
                for (uint32_t l = x * kLate / kSpread; l < kLate && l < (x + 1) * kLate / kSpread; ++l) issue(kb + SLOTS - 1, before, kEarly + l, gone_before);
            } else {
                if (j == 0) b[0] = fragment(next_at + b_lo, 0);
                a[j] = fragment(next_at + a_lo, j);
                if (j < kEarly) issue(kb + SLOTS, slot, j, gone_here);
                if constexpr (ROW_SCALES)
                    if (j == FM - 1) row_scales(next_scales, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (uint32_t x = FN * FM - 3; x < FN * FM; ++x) add(x);
        if (in_span == kPlace && more) place_scales(span + 1);
#pragma unroll
        for (uint32_t j = 0; j < FM; ++j) s[j] = ROW_SCALES ? s_next[j] : s_next[j] * sb;
        slot = next;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // the loads past the end, before the LDS changes hands
    if (p.parts != nullptr) {
        float* const part = p.parts + (size_t)blockIdx.y * p.m * p.n_wide;
#pragma unroll
        for (uint32_t j = 0; j < FM; ++j) {
            const uint32_t row = wm * (TM / WM) + 16 * j + r16;
#pragma unroll
            for (uint32_t i = 0; i < FN; ++i) {
                const uint32_t n = n0 + wn * (TN / WN) + 16 * i + 4 * quarter;
                if (row < w.rows && n < p.n) *reinterpret_cast<v4f*>(part + (size_t)(w.row0 + row) * p.n_wide + n) = sum[i][j];
            }
        }
        return;
    }
    const uint32_t size = p.out_type == CMX_OUT_FP32 ? 4 : 2;
#pragma unroll
    for (uint32_t j = 0; j < FM; ++j) {
        const uint32_t row = wm * (TM / WM) + 16 * j + r16;
        uint8_t* const c_row = p.c + (size_t)(w.row0 + row) * p.ldc * size;
#pragma unroll
        for (uint32_t i = 0; i < FN; ++i) {
            const uint32_t n = n0 + wn * (TN / WN) + 16 * i + 4 * quarter;
            if (row < w.rows && n < p.n) store4(c_row, n, sum[i][j], p.out_type, p.n - n);
        }
    }
}

// the parts of every sum, in the order of K
__global__ __launch_bounds__(256) void fp8_join_kernel(const Fp8GemmArgs p, uint32_t splits) {
    const uint32_t quads = p.n_wide / 4, item = blockIdx.x * 256 + threadIdx.x, row = item / quads, n = 4 * (item - row * quads);
    if (row >= p.m) return;
    const v4f* part = reinterpret_cast<const v4f*>(p.parts) + item;
    const size_t step = (size_t)p.m * quads;
    v4f sum = {0, 0, 0, 0};
    for (uint32_t s0 = 0; s0 < splits; s0 += 4) {
        v4f v[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = s0 + i < splits ? part[(s0 + i) * step] : (v4f){0, 0, 0, 0};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) sum += v[i];
    }
    store4(p.c + (size_t)row * p.ldc * (p.out_type == CMX_OUT_FP32 ? 4 : 2), n, sum, p.out_type, p.n - n);
}

// m-tiles of TM rows that a launch may need: the groups' own, and those of the rows behind them
uint64_t most_tiles(const Fp8GemmArgs& p, uint32_t tm) {
    if (p.sizes == nullptr) return ceil_div(p.m, tm);
    return p.m / tm + std::min(p.groups, p.m) + 1;
}

template <int FMT, int FN, int FM, int DEPTH, bool ROW_SCALES>
int launch_rows(Fp8GemmArgs p, hipStream_t s, uint32_t most_waves) {
    p.n_tiles = ceil_div(p.n, 16 * FN);
    const uint64_t tiles = most_tiles(p, 16 * FM) * p.n_tiles;
    // as many wavefronts as share the blocks of K evenly
    const uint32_t waves = ceil_div(p.blocks, ceil_div(p.blocks, most_waves));
    CMX_REQUIRE(fits_grid(tiles, 64 * waves), "too many tiles");
    // operands of a wavefront on their way into fragments, then its sums
    constexpr size_t kEach = std::max(FN * FM * 64 * 16, (FN + FM) * 16 * (int)kBlockK);
    constexpr size_t kMost = (FN * FM == 1 ? 16 : 8) * kEach;
    if constexpr (kMost > 64 * 1024)
        if (int rc = allow_dynamic_lds<fp8_rows_kernel<FMT, FN, FM, DEPTH, ROW_SCALES>, kMost>(); rc != CMX_OK) return rc;
    hipLaunchKernelGGL((fp8_rows_kernel<FMT, FN, FM, DEPTH, ROW_SCALES>), dim3((uint32_t)tiles), dim3(64 * waves), waves * kEach, s, p);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

template <int FMT, int TN, int TM, int WN, int WM, int SLOTS, bool ROW_SCALES>
int launch_tile(Fp8GemmArgs p, hipStream_t s, uint32_t splits = 1) {
    constexpr auto kfn = fp8_tile_kernel<FMT, TN, TM, WN, WM, SLOTS, ROW_SCALES>;
    constexpr size_t smem = SLOTS * (TN + TM) * kBlockK + 2 * (TM + (ROW_SCALES ? TN : 0)) * kSpanOf<ROW_SCALES> * 4 + (SLOTS == 2 ? 512 : 0);
    static_assert(smem <= 160 * 1024, "LDS");
    if (int rc = allow_dynamic_lds<kfn, smem>(); rc != CMX_OK) return rc;
    p.n_tiles = ceil_div(p.n, TN);
    const uint64_t tiles = most_tiles(p, TM) * p.n_tiles;
    CMX_REQUIRE(fits_grid(tiles, 64 * WN * WM), "too many tiles");
    if (splits > 1) {
        p.split_blocks = ceil_div(p.blocks, splits);
        splits = ceil_div(p.blocks, p.split_blocks);
        p.n_wide = round_up(p.n, 4);
    } else {
        p.parts = nullptr;
    }
    hipLaunchKernelGGL(kfn, dim3((uint32_t)tiles, splits), dim3(64 * WN * WM), smem, s, p);
    CMX_LAUNCH_CHECK();
    if (splits > 1) {
        hipLaunchKernelGGL(fp8_join_kernel, dim3(ceil_div(p.m * (p.n_wide / 4), 256)), dim3(256), 0, s, p, splits);
        CMX_LAUNCH_CHECK();
    }
    return CMX_OK;
}

// How a product is computed: the kernel and, for a dense one of few tiles, how many workgroups share the K of a tile.
enum class Way { kRows1x1, kRows4x1, kRows1x2, kRows2x2, kRows2x4, kTile128, kTile256x128, kTile256 };
struct Plan {
    Way way;
    uint32_t splits, waves;
};

// The way that a model of its time says is the shortest.  A workgroup takes `start` + `block` * blocks us where one runs on each CU, as measured with 256 of them
// (`block` holds for the whole chip's share of memory, too):
//                                us, start + block * blocks          measured, 8 and 56 blocks of K
//   rows, 16 x 16 a wavefront    2.3 + 0.09                          1 x 4096: 3.0, 7.3;   in 64 x 16: 6.5 (56)
//   rows, 64 x 16                2 + 0.36                            1 x 16384: 4.8, 22.1; in 16 x 16: 5.4, 26
//   rows, 16 x 32                2.5 + 0.127                         32 x 4096: 3.5, 9.6
//   rows, 32 x 32                2.3 + 0.185                         64 x 4096: 3.8, 12.7; in 16 x 32: 4.4, 16.2
//   rows, 32 x 64                3.2 + 0.24                          128 x 4096: 5.1, 16.8; in 32 x 32: 7.0, 22.8
//   tile 128 x 128               4.5 + 0.61                          1024 x 4096: 38.4 (56); in 256 x 128: 54
//   tile 256 x 128               5 + 1.05                            2048 x 4096: 59.6 (56); in 128 x 128: 77, in 256 x 256: 84
//   tile 256 x 256               6 + 1.75                            8192 x 4096: 210 (56, two rounds); in 256 x 128: 243
// Both sides of a border are from one run; other runs are up to a tenth longer (8192 x 4096 x 7168 216 - 224).  All with a scale for 128 rows of b: with one for every row the same rule holds, for
// which no borders were measured (4096 x 2048 x 2784 then takes a fifth longer, 64 x 4096 x 7168 a tenth).
// Workgroups of the rows kernel follow each other without a gap, those of the tiles come in rounds.  A tile's K is split over workgroups where there are few: 3 us for
// the launch that joins them, and twice their sums' way through memory (256 x 4096 x 7168 four ways 21, in one piece 41, by rows of 32 x 64 31).  Groups whose rows fit one tile are bound by their
// weights, which rows of 64 x 16 read at 0.9 of a stream's rate and the tiles
// at 0.75, 256 x 128 the best (64 groups of 8 rows, 4096 x 2048: rows 95 us, 256 x 128 106; of 24: 256 x 128 110, 128 x 128 125, 256 x 256 144).
Plan plan_of(const Fp8GemmArgs& p, uint32_t cus, bool may_split) {
    const bool grouped = p.sizes != nullptr;
    // groups that have rows, where rows fall on them at random
    const double used = grouped ? p.groups * (1.0 - std::exp(p.groups > 1 ? p.m * std::log1p(-1.0 / p.groups) : -1e9)) : 1.0;
    const double blocks = p.blocks;
    const double stream = used * p.n * (double)p.k / 6.1e6;            // us that reading the weights takes
    // (groups well below a tile are one each, others end half a tile behind their rows on average)
    const auto m_tiles = [&](uint32_t tm) -> double {
        if (!grouped) return ceil_div(p.m, tm);
        return p.m <= 0.8 * tm * used ? used : p.m / (double)tm + used / 2;
    };
    Plan best{Way::kTile128, 1, 0};
    double least = 1e300;
    const auto offer = [&](Way way, double us, uint32_t splits, uint32_t waves) {
        if (us < least) {
            least = us;
            best = {way, splits, waves};
        }
    };
    const auto rows = [&](Way way, uint32_t tn, uint32_t tm, double start, double block, uint32_t waves) {
        const double groups = m_tiles(tm) * ceil_div(p.n, tn) / cus;
        // (a workgroup that looks for its group takes 1.2 us more)
        offer(way, std::max(start + block * blocks * std::max(groups, 1.0) + (grouped ? 1.2 * std::max(groups - 1.0, 0.0) : 0.0), 1.1 * stream + 3), 1, way == Way::kRows4x1 || way == Way::kRows2x2 ? (groups >= 2 ? 4 : 8) : waves);
    };
    rows(Way::kRows1x1, 16, 16, 2.3, 0.09, 16);
    rows(Way::kRows4x1, 64, 16, 2.0, 0.36, 8);
    rows(Way::kRows1x2, 16, 32, 2.5, 0.127, 8);
    rows(Way::kRows2x2, 32, 32, 2.3, 0.185, 8);
    rows(Way::kRows2x4, 32, 64, 3.2, 0.24, 8);
    const auto tile = [&](Way way, uint32_t tn, uint32_t tm, double start, double block) {
        const double rounds = std::ceil(m_tiles(tm) * ceil_div(p.n, tn) / cus);
        offer(way, std::max(start + block * blocks * rounds, 1.3 * stream + 4), 1, 0);
    };
    tile(Way::kTile256x128, 256, 128, 5.0, 1.05);
    tile(Way::kTile128, 128, 128, 4.5, 0.61);
    tile(Way::kTile256, 256, 256, 6.0, 1.75);
    if (!grouped && may_split && p.m > 16) {                          // (ops.py knows that fewer rows, and fewer than 8 blocks, are not split)
        const uint64_t tiles = (uint64_t)ceil_div(p.m, 128) * ceil_div(p.n, 128);
        const uint32_t splits = (uint32_t)std::min<uint64_t>({cus / std::max<uint64_t>(tiles, 1), 16, p.blocks / 4});
        if (splits > 1) {
            const double sums = splits * (double)p.m * p.n * 8 / 4.5e6;
            offer(Way::kTile128, std::max(4.5 + 0.61 * std::ceil(blocks / splits), 1.3 * stream + 4) + 3 + sums, splits, 0);
        }
    }
    return best;
}

size_t parts_bytes(const Fp8GemmArgs& p, const Plan& plan) { return plan.splits > 1 ? (size_t)plan.splits * p.m * round_up(p.n, 4) * sizeof(float) : 0; }

template <int FMT, bool ROW_SCALES>
int launch(const Fp8GemmArgs& p, hipStream_t s) {
    int cus;
    if (int rc = cu_count(&cus); rc != CMX_OK) return rc;
    const Plan plan = plan_of(p, cus, p.parts != nullptr);
    switch (plan.way) {
        case Way::kRows1x1: return launch_rows<FMT, 1, 1, 2, ROW_SCALES>(p, s, plan.waves);
        case Way::kRows4x1: return launch_rows<FMT, 4, 1, 2, ROW_SCALES>(p, s, plan.waves);
        case Way::kRows1x2: return launch_rows<FMT, 1, 2, 2, ROW_SCALES>(p, s, plan.waves);
        case Way::kRows2x2: return launch_rows<FMT, 2, 2, 2, ROW_SCALES>(p, s, plan.waves);
        case Way::kRows2x4: return launch_rows<FMT, 2, 4, 1, ROW_SCALES>(p, s, plan.waves);
        case Way::kTile128: return launch_tile<FMT, 128, 128, 4, 2, 3, ROW_SCALES>(p, s, plan.splits);
        case Way::kTile256x128: return launch_tile<FMT, 256, 128, 4, 2, 3, ROW_SCALES>(p, s);
        case Way::kTile256: return launch_tile<FMT, 256, 256, 2, 4, 2, ROW_SCALES>(p, s);
    }
    return CMX_EINVAL;
}

int fp8_block_product(const Fp8GemmArgs& p, int fmt, uint32_t b_rows, hipStream_t s) {
    if (fmt == CMX_FMT_E5M2) return b_rows == 1 ? launch<CMX_FMT_E5M2, true>(p, s) : launch<CMX_FMT_E5M2, false>(p, s);
    return b_rows == 1 ? launch<CMX_FMT_E4M3, true>(p, s) : launch<CMX_FMT_E4M3, false>(p, s);
}

int check_product(const Fp8GemmArgs& p, const void* c, int fmt) {
    CMX_REQUIRE(fmt == CMX_FMT_E4M3 || fmt == CMX_FMT_E5M2, "8-bit formats only");
    CMX_REQUIRE(p.out_type == CMX_OUT_BF16 || p.out_type == CMX_OUT_FP16 || p.out_type == CMX_OUT_FP32, "unknown type");
    if (p.m == 0 || p.n == 0) return CMX_OK;
    CMX_REQUIRE(p.a && p.a_scale && p.b && p.b_scale && c, "null pointer");
    CMX_REQUIRE(p.k > 0 && p.k % 16 == 0, "k must be a positive multiple of 16");
    CMX_REQUIRE(p.m < (1u << 31) && p.n < (1u << 31), "at most 2^31 - 1 rows and columns");
    CMX_REQUIRE(p.lda >= p.k && p.ldb >= p.k && p.ld_as >= p.blocks && p.ld_bs >= p.blocks && p.ldc >= p.n, "row pitch smaller than row");
    CMX_REQUIRE(aligned16(p.a) && aligned16(p.b) && p.lda % 16 == 0 && p.ldb % 16 == 0, "operand rows must be 16-byte aligned");
    CMX_REQUIRE(reinterpret_cast<uintptr_t>(p.a_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(p.b_scale) % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(c) % (p.out_type == CMX_OUT_FP32 ? 4 : 2) == 0, "pointers must be aligned to their elements");
    CMX_REQUIRE(p.lda <= (1u << 22) && p.ldb <= (1u << 22), "operand rows may be at most 2^22 bytes apart");      // (offsets in a tile stay below 2^31)
    return CMX_OK;
}

}  // namespace
}  // namespace cmx

int cmx::preload_fp8_gemm_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::fp8_rows_kernel<CMX_FMT_E4M3, 1, 1, 2, false>)));
    return CMX_OK;
}

#ifdef CMX_TEST_HOOKS
// the way of a product on a chip of `cus` CUs: Way, and 256 times its parts of K; groups = 0: dense
extern "C" int cmx_debug_fp8_way(uint32_t m, uint32_t n, uint32_t k, uint32_t groups, int workspace, uint32_t cus) {
    using namespace cmx;
    const int32_t sizes = 0;
    Fp8GemmArgs p{};
    p.m = m;
    p.n = n;
    p.k = k;
    p.blocks = ceil_div(k, kBlockK);
    p.groups = groups;
    p.sizes = groups != 0 ? &sizes : nullptr;
    const Plan plan = plan_of(p, cus, workspace != 0);
    return (int)plan.way | (int)plan.splits << 8;
}
#endif

extern "C" size_t cmx_fp8_block_gemm_workspace_bytes(uint32_t m, uint32_t n, uint32_t k) {
    using namespace cmx;
    if (m == 0 || n == 0 || k == 0) return 0;
    int cus;
    if (cu_count(&cus) != CMX_OK) cus = 256;
    Fp8GemmArgs p{};
    p.m = m;
    p.n = n;
    p.k = k;
    p.blocks = ceil_div(k, kBlockK);
    return parts_bytes(p, plan_of(p, cus, true));
}

extern "C" int cmx_fp8_block_gemm(const uint8_t* a, uint32_t lda, const float* a_scale, uint32_t ld_as, const uint8_t* b, uint32_t ldb, const float* b_scale,
                                  uint32_t ld_bs, uint32_t b_rows, void* c, uint32_t ldc, uint32_t m, uint32_t n, uint32_t k, int fmt, int out_type,
                                  void* workspace, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(b_rows == 1 || b_rows == 128, "b has a scale for every row or every 128 rows");
    const Fp8GemmArgs p = {a, b, a_scale, b_scale, static_cast<uint8_t*>(c), nullptr, 0, 0, lda, ldb, ld_as, ld_bs, ldc, m, n, k, ceil_div(k, kBlockK), 1, 0, 0, out_type,
                           static_cast<float*>(workspace), 0, 0};
    if (int rc = check_product(p, c, fmt); rc != CMX_OK || m == 0 || n == 0) return rc;
    CMX_REQUIRE(aligned16(workspace), "the workspace must be 16-byte aligned");
    return fp8_block_product(p, fmt, b_rows, static_cast<hipStream_t>(stream));
}

extern "C" int cmx_fp8_block_gmm(const uint8_t* a, uint32_t lda, const float* a_scale, uint32_t ld_as, const uint8_t* b, const float* b_scale, void* c,
                                 uint32_t ldc, const int32_t* group_sizes, uint32_t groups, uint32_t m_total, uint32_t n, uint32_t k, int fmt, int out_type,
                                 int zero_rest, cmx_stream_t stream) {
    using namespace cmx;
    const uint32_t blocks = ceil_div(k, kBlockK);
    const Fp8GemmArgs p = {a, b, a_scale, b_scale, static_cast<uint8_t*>(c), group_sizes, (size_t)n * k, (size_t)ceil_div(n, 128) * blocks, lda, k, ld_as, blocks, ldc,
                           m_total, n, k, blocks, groups, 0, zero_rest ? 1u : 0u, out_type, nullptr, 0, 0};
    if (groups == 0 && !zero_rest) return CMX_OK;
    if (int rc = check_product(p, c, fmt); rc != CMX_OK || m_total == 0 || n == 0) return rc;
    CMX_REQUIRE(group_sizes != nullptr, "null pointer");
    CMX_REQUIRE(groups > 0 && groups <= (1u << 20), "between 1 and 2^20 groups");
    return fp8_block_product(p, fmt, 128, static_cast<hipStream_t>(stream));
}
