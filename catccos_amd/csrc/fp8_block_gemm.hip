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

// ---- few rows ------------------------------------------------------------------------------------------------------------
// A workgroup owns 16 FN columns of c and 16 FM rows over all of K; its wavefronts take the blocks of K in turn, DEPTH of each in flight, and join their
// sums in LDS in the order of the wavefronts.  Lane l holds row l % 16 of an operand, the 16-byte pieces l / 16 and l / 16 + 4 of a block.
template <int FMT, int FN, int FM, int DEPTH, bool ROW_SCALES>
__global__ __launch_bounds__(512) void fp8_rows_kernel(const Fp8GemmArgs p) {
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
    const uint8_t *b_row[FN], *a_row[FM];
    const float *b_scale[FN], *a_scale[FM];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        const uint32_t n = min(n0 + 16 * i + r16, p.n - 1);
        b_row[i] = p.b + w.g * p.b_step + (size_t)n * p.ldb;
        b_scale[i] = p.b_scale + w.g * p.bs_step + (ROW_SCALES ? (size_t)min(n0 + 16 * i + 4 * quarter, p.n - 1) * p.ld_bs : (size_t)((n0 + 16 * i) / kBlockK) * p.ld_bs);
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const uint32_t m = w.row0 + min(16 * j + r16, w.rows - 1);
        a_row[j] = p.a + (size_t)m * p.lda;
        a_scale[j] = p.a_scale + (size_t)m * p.ld_as;
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
    const bool lo_in = tail == 0 || 16 * quarter < tail, hi_in = tail == 0 || 16 * quarter + 64 < tail;
    const auto whole = [&](const uint8_t* row, uint32_t kb) -> v8i {
        const uint32_t at = kb * kBlockK + 16 * quarter;
        const v4i lo = *reinterpret_cast<const v4i*>(row + min(at, far)), hi = *reinterpret_cast<const v4i*>(row + min(at + 64, far));
        return (v8i){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    const auto cleared = [&](v8i& v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = lo_in ? v[i] : 0;
            v[4 + i] = hi_in ? v[4 + i] : 0;
        }
    };
    for (uint32_t kb0 = wave; kb0 < p.blocks; kb0 += DEPTH * waves) {
        v8i b[DEPTH][FN], a[DEPTH][FM];
        float sb[DEPTH][FN][ROW_SCALES ? 4 : 1], sa[DEPTH][FM];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const uint32_t kb = kb0 + d * waves;
            if (kb >= p.blocks) break;
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                b[d][i] = whole(b_row[i], kb);
                if constexpr (ROW_SCALES) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) sb[d][i][r] = b_scale[i][(size_t)bs_at[i][r] * p.ld_bs + kb];
                } else {
                    sb[d][i][0] = b_scale[i][kb];
                }
            }
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                a[d][j] = whole(a_row[j], kb);
                sa[d][j] = a_scale[j][kb];
            }
        }
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (kb0 + d * waves >= p.blocks) break;
            if (tail != 0 && kb0 + d * waves == last) {
#pragma unroll
                for (int i = 0; i < FN; ++i) cleared(b[d][i]);
#pragma unroll
                for (int j = 0; j < FM; ++j) cleared(a[d][j]);
            }
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j) {
                    const v4f part = block_product<FMT>(b[d][i], a[d][j]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum[i][j][r] = __builtin_fmaf(part[r], sa[d][j] * sb[d][i][ROW_SCALES ? r : 0], sum[i][j][r]);
                }
        }
    }
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
// A workgroup of WN x WM wavefronts owns TN columns and TM rows of c.  Blocks of K travel by LDS-DMA into SLOTS slots; row r of a slot holds its 16-byte piece p at
// place p ^ (r / 2 % 8), so that the 16 rows that a fragment reads at a time lie in different banks.
__device__ __forceinline__ uint32_t place_of(uint32_t row, uint32_t piece) { return piece ^ ((row >> 1) & 7u); }
__device__ __forceinline__ uint32_t same(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ void dma16(uint32_t lds, uint32_t off, v4i rsrc, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(same(lds)), "v"(off), "s"(rsrc), "s"(same(soff)) : "memory");
}
__device__ __forceinline__ v4i buffer_at(const uint8_t* base) {
    const uint64_t v = reinterpret_cast<uint64_t>(base);
    return (v4i){(int)same((uint32_t)v), (int)same((uint32_t)(v >> 32)), (int)0x80000000u, 0x00020000};      // offsets of 2^31 on give zeros
}

constexpr uint32_t kScaleSpan = 8;                    // blocks of K whose scales lie in LDS at a time (twice)

template <int FMT, int TN, int TM, int WN, int WM, int SLOTS, bool ROW_SCALES>
__global__ __launch_bounds__(64 * WN * WM) void fp8_tile_kernel(const Fp8GemmArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr uint32_t NW = WN * WM, NT = 64 * NW, FN = TN / WN / 16, FM = TM / WM / 16, kRows = TN + TM, kSlot = kRows * kBlockK;
    constexpr uint32_t kLoads = kRows / (8 * NW), kBLoads = TN / (8 * NW);
    constexpr uint32_t kScaleRows = TM + (ROW_SCALES ? TN : 0), kScaleBase = SLOTS * kSlot, kScaleHalf = kScaleRows * kScaleSpan * 4;
    static_assert(TN % (8 * NW) == 0 && TM % (8 * NW) == 0 && (8 * NW) % 16 == 0, "loads of whole rows, the same piece in all of a lane's");
    static_assert(128 % (TN / WN) == 0, "a wavefront's columns share a scale");
    static_assert(2 * kLoads <= FN * FM && FM >= 3, "loads behind every other product; a fragment of b is free again when its last sums are added");
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
    // scales of blocks span * kScaleSpan .. + kScaleSpan, [block][row], into half span % 2; a thread has some rows' four blocks
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

    fetch_scales(0);
    place_scales(0);
#pragma unroll
    for (uint32_t d = 0; d + 1 < SLOTS; ++d)
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) issue(d, d, i, gone(d));
    uint32_t slot = 0;
    float sb = ROW_SCALES ? 0.0f : b_scale[0];
    for (uint32_t kb = 0; kb < p.blocks; ++kb) {
        // block kb has arrived for all, and all have read block kb - 1
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((SLOTS - 2) * kLoads) : "memory");
        const uint32_t next_slot = slot == 0 ? SLOTS - 1 : slot - 1, next_gone = gone(kb + SLOTS - 1);
        const uint32_t span = kb / kScaleSpan, in_span = kb % kScaleSpan;
        const bool more = (span + 1) * kScaleSpan < p.blocks;
        if (in_span == 1 && more) fetch_scales(span + 1);
        const uint32_t at = lds0 + slot * kSlot;
        const float* const scales = reinterpret_cast<const float*>(smem + kScaleBase + (span & 1u) * kScaleHalf) + in_span * kScaleRows;
        v8i a[FM], b[2];
        float s[FM];
        v4f part[4], rs[3];
        const uint32_t b_row = wn * (TN / WN), a_row = wm * (TM / WM) + r16, b_at = at + b_lo, a_at = at + a_lo;
        const auto b_fragment = [&](uint32_t i) {
            b[i & 1] = fragment(b_at, i);
            if constexpr (ROW_SCALES) rs[i % 3] = *reinterpret_cast<const v4f*>(scales + TM + b_row + 16 * i + 4 * quarter);
        };
        b_fragment(0);
#pragma unroll
        for (uint32_t j = 0; j < FM; ++j) {
            a[j] = fragment(a_at, j);
            s[j] = scales[a_row + 16 * j];
            if constexpr (!ROW_SCALES) s[j] *= sb;
        }
        __builtin_amdgcn_sched_barrier(0);
        const auto add = [&](uint32_t x) {
            const uint32_t i = x / FM, j = x % FM;
            asm volatile("" : "+v"(part[x % 4]));                      // (not in AGPRs, from which the vector unit would have to copy it)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (ROW_SCALES) sum[i][j][r] = __builtin_fmaf(part[x % 4][r], rs[i % 3][r] * s[j], sum[i][j][r]);
                else sum[i][j][r] = __builtin_fmaf(part[x % 4][r], s[j], sum[i][j][r]);
            }
            asm volatile("" : "+v"(sum[i][j]));                        // (used here: the compiler would put all multiply-adds behind all products)
        };
        // a product, the multiply-adds of the one three before, its share of the loads: in this order
#pragma unroll
        for (uint32_t x = 0; x < FN * FM; ++x) {
            part[x % 4] = block_product<FMT>(b[x / FM & 1], a[x % FM]);
            if (x >= 3) add(x - 3);
            if (x % FM == 0 && x / FM + 1 < FN) b_fragment(x / FM + 1);
            if (x % 2 == 1 && x / 2 < kLoads) issue(kb + SLOTS - 1, next_slot, x / 2, next_gone);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (uint32_t x = FN * FM - 3; x < FN * FM; ++x) add(x);
        if (in_span == 4 && more) place_scales(span + 1);
        if constexpr (!ROW_SCALES) sb = b_scale[min(kb + 1, last)];
        slot = slot + 1 < SLOTS ? slot + 1 : 0;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // the loads past the end, before the LDS changes hands
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

// m-tiles of TM rows that a launch may need: the groups' own, and those of the rows behind them
uint64_t most_tiles(const Fp8GemmArgs& p, uint32_t tm) {
    if (p.sizes == nullptr) return ceil_div(p.m, tm);
    return p.m / tm + std::min(p.groups, p.m) + 1;
}

template <int FMT, int FN, int FM, int DEPTH, bool ROW_SCALES>
int launch_rows(Fp8GemmArgs p, hipStream_t s) {
    p.n_tiles = ceil_div(p.n, 16 * FN);
    const uint64_t tiles = most_tiles(p, 16 * FM) * p.n_tiles;
    const uint32_t waves = std::min(8u, p.blocks);
    CMX_REQUIRE(fits_grid(tiles, 64 * waves), "too many tiles");
    constexpr size_t kEach = FN * FM * 64 * 16;
    static_assert(8 * kEach <= 64 * 1024, "LDS");
    hipLaunchKernelGGL((fp8_rows_kernel<FMT, FN, FM, DEPTH, ROW_SCALES>), dim3((uint32_t)tiles), dim3(64 * waves), waves * kEach, s, p);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

template <int FMT, int TN, int TM, int WN, int WM, int SLOTS, bool ROW_SCALES>
int launch_tile(Fp8GemmArgs p, hipStream_t s) {
    constexpr auto kfn = fp8_tile_kernel<FMT, TN, TM, WN, WM, SLOTS, ROW_SCALES>;
    constexpr size_t smem = SLOTS * (TN + TM) * kBlockK + 2 * (TM + (ROW_SCALES ? TN : 0)) * kScaleSpan * 4;
    static_assert(smem <= 160 * 1024, "LDS");
    if (int rc = allow_dynamic_lds<kfn, smem>(); rc != CMX_OK) return rc;
    p.n_tiles = ceil_div(p.n, TN);
    const uint64_t tiles = most_tiles(p, TM) * p.n_tiles;
    CMX_REQUIRE(fits_grid(tiles, 64 * WN * WM), "too many tiles");
    hipLaunchKernelGGL(kfn, dim3((uint32_t)tiles), dim3(64 * WN * WM), smem, s, p);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

template <int FMT, bool ROW_SCALES>
int launch(const Fp8GemmArgs& p, hipStream_t s) {
    int cus;
    if (int rc = cu_count(&cus); rc != CMX_OK) return rc;
    const uint32_t rows = p.sizes == nullptr ? p.m : ceil_div(p.m, std::max(1u, std::min(p.groups, p.m)));      // of a group, on average
    if (rows <= 16) return launch_rows<FMT, 1, 1, 4, ROW_SCALES>(p, s);
    if (rows <= 64) return launch_rows<FMT, 1, 4, 2, ROW_SCALES>(p, s);
    if (most_tiles(p, 256) * ceil_div(p.n, 256) >= (uint32_t)cus && rows > 128) return launch_tile<FMT, 256, 256, 2, 4, 2, ROW_SCALES>(p, s);
    return launch_tile<FMT, 128, 128, 2, 2, 3, ROW_SCALES>(p, s);
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
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::fp8_rows_kernel<CMX_FMT_E4M3, 1, 1, 4, false>)));
    return CMX_OK;
}

extern "C" int cmx_fp8_block_gemm(const uint8_t* a, uint32_t lda, const float* a_scale, uint32_t ld_as, const uint8_t* b, uint32_t ldb, const float* b_scale,
                                  uint32_t ld_bs, uint32_t b_rows, void* c, uint32_t ldc, uint32_t m, uint32_t n, uint32_t k, int fmt, int out_type,
                                  cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(b_rows == 1 || b_rows == 128, "b has a scale for every row or every 128 rows");
    const Fp8GemmArgs p = {a, b, a_scale, b_scale, static_cast<uint8_t*>(c), nullptr, 0, 0, lda, ldb, ld_as, ld_bs, ldc, m, n, k, ceil_div(k, kBlockK), 1, 0, 0, out_type};
    if (int rc = check_product(p, c, fmt); rc != CMX_OK || m == 0 || n == 0) return rc;
    return fp8_block_product(p, fmt, b_rows, static_cast<hipStream_t>(stream));
}

extern "C" int cmx_fp8_block_gmm(const uint8_t* a, uint32_t lda, const float* a_scale, uint32_t ld_as, const uint8_t* b, const float* b_scale, void* c,
                                 uint32_t ldc, const int32_t* group_sizes, uint32_t groups, uint32_t m_total, uint32_t n, uint32_t k, int fmt, int out_type,
                                 int zero_rest, cmx_stream_t stream) {
    using namespace cmx;
    const uint32_t blocks = ceil_div(k, kBlockK);
    const Fp8GemmArgs p = {a, b, a_scale, b_scale, static_cast<uint8_t*>(c), group_sizes, (size_t)n * k, (size_t)ceil_div(n, 128) * blocks, lda, k, ld_as, blocks, ldc,
                           m_total, n, k, blocks, groups, 0, zero_rest ? 1u : 0u, out_type};
    if (groups == 0 && !zero_rest) return CMX_OK;
    if (int rc = check_product(p, c, fmt); rc != CMX_OK || m_total == 0 || n == 0) return rc;
    CMX_REQUIRE(group_sizes != nullptr, "null pointer");
    CMX_REQUIRE(groups > 0 && groups <= (1u << 20), "between 1 and 2^20 groups");
    return fp8_block_product(p, fmt, 128, static_cast<hipStream_t>(stream));
}
