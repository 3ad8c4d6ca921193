// E4M3 / E5M2 codes with an fp32 scale for each block of 128 (1 x 128, or 128 x 128) of a matrix or of its transpose.
//
//   s = max(max |z| / most, 2^-126), or the least power of two that is no less;  code = the nearest value to z / s, ties to even
//
// The quotient is that of the exact z / s, not of its fp32 value.
// Bound by memory: 3 bytes to a 16-bit element.
#include <type_traits>

#include "mx_launch.h"

namespace cmx {
namespace {

constexpr uint32_t kBlock = 128;
constexpr float kLeastScale = 1.17549435e-38f;       // 2^-126
constexpr uint32_t kInfBits = 0x7F800000u;

struct Fp8QuantArgs {
    const uint8_t* x;
    uint8_t* codes;
    float* scales;
    size_t ld_x, x_step;                             // bytes
    uint32_t ld_codes, ld_scales;
    uint32_t rows, cols;                             // of x
    uint32_t out_cols, out_wide;                     // of the codes: without and with the zeros behind a row
    uint32_t out_rows, scale_rows, blocks;
    uint32_t vec;                                    // rows of x are whole 16-byte pieces
    uint32_t pow2;
    uint32_t block_part;                             // 65536 / blocks, rounded up, for few blocks
};

template <bool STREAM, class V>
__device__ __forceinline__ V load_piece(const uint8_t* p, uint32_t i = 0) {
    return STREAM ? __builtin_nontemporal_load(reinterpret_cast<const V*>(p) + i) : reinterpret_cast<const V*>(p)[i];
}

// eight consecutive elements of type T, `n` of them there, the others zero
template <int TYPE, bool STREAM = false>
__device__ __forceinline__ void load8(const uint8_t* p, bool whole, uint32_t n, float (&v)[8]) {
    if constexpr (TYPE == CMX_OUT_FP32) {
        if (whole) {
            const v4f lo = load_piece<STREAM, v4f>(p), hi = load_piece<STREAM, v4f>(p, 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) v[i] = i < n ? reinterpret_cast<const float*>(p)[i] : 0.0f;
        }
        return;
    }
    uint32_t w[4];
    if (whole) {
        const v4i d = load_piece<STREAM, v4i>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)d[i];
    } else {
        const uint16_t* const h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) w[i] = (2 * i < n ? h[2 * i] : 0u) | ((2 * i + 1 < n ? (uint32_t)h[2 * i + 1] : 0u) << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == CMX_OUT_BF16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
            v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
        }
    }
}

// bits of |v| order like the values, with Inf above them and NaN above that
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

template <int FMT>
struct BlockScale {
    float s, inverse;
    bool finite;
    __device__ __forceinline__ BlockScale(uint32_t amax_bits, uint32_t pow2) {
        constexpr float kMost = FMT == CMX_FMT_E5M2 ? 57344.0f : 448.0f, kPart = 1.0f / kMost;
        finite = amax_bits < kInfBits;
        const float amax = __uint_as_float(amax_bits);
        s = amax;                                                     // (Inf and NaN are scales themselves)
        if (finite) {
            // the quotient rounded to nearest: what amax * (1 / most) is off by is known exactly, and small
            s = amax * kPart;
            s = __builtin_fmaf(__builtin_fmaf(-s, kMost, amax), kPart, s);
            // amax / most is no closer above a power of two than its fp32 quotient can tell: 448 and 57344 are 1.75 * 2^i, and of the amax right above
            // such a value the quotient is 1 + 2^-23 / 1.75
            if (pow2) s = __uint_as_float((__float_as_uint(s) + 0x007FFFFFu) & 0xFF800000u);
            s = fmaxf(s, kLeastScale);
        }
        inverse = __builtin_amdgcn_rcpf(s);
    }
    __device__ __forceinline__ BlockScale(float scale, float inv, bool is_finite) : s(scale), inverse(inv), finite(is_finite) {}
};

template <int FMT>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    uint32_t w = 0;
    if constexpr (FMT == CMX_FMT_E5M2) {
        w = cvt_pk_e5m2(a, b, w, false);
        return cvt_pk_e5m2(c, d, w, true);
    }
    w = cvt_pk_e4m3(a, b, w, false);
    return cvt_pk_e4m3(c, d, w, true);
}

// z into numbers that the hardware's cast rounds to the codes of the exact z / s.  Codes and the borders between them have at most 5 significant bits (E5M2 4): b is the value
// of so many bits that z * (1 / s) is next to, and if z / s is not b it lies on the side of b that the sign of z - b * s says, one fused multiply-add; the cast gets b
// moved to that side by 2^-10 of itself, which crosses nothing.  (z - b * s is a multiple of 2^-28 of z, so that 2^30 times it exceeds the 2^-10.)
// 8 operations an element for all of them: a look for values next to a border first takes 5, but of bf16 elements so many lie on one (3/4 and 3/2 of a maximum are borders) that
// two wavefronts in five went on (8192 x 7168: 25 vector operations an element and 35.6 us, so 33).
template <int FMT, int N>
__device__ __forceinline__ void quotients(float (&z)[N], BlockScale<FMT> b) {
    constexpr uint32_t kUnder = FMT == CMX_FMT_E5M2 ? 20 : 19;
    if (b.s < 0x1p-60f) {                                              // (what is left of a small z would lie below fp32's least value)
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] *= 0x1p100f;
        b.s *= 0x1p100f;
        b.inverse *= 0x1p-100f;
    }
    const float far = b.inverse * 0x1p30f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float q = __uint_as_float((__float_as_uint(z[i] * b.inverse) + (1u << (kUnder - 1))) & ~((1u << kUnder) - 1)), step = fabsf(q) * 0x1p-10f;
        z[i] = q + __builtin_amdgcn_fmed3f(__builtin_fmaf(-q, b.s, z[i]) * far, -step, step);
    }
}

template <int FMT>
__device__ __forceinline__ uint2 codes8(float (&z)[8], const BlockScale<FMT>& b) {
    if (!b.finite) return make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
    quotients<FMT>(z, b);
    return make_uint2(codes4<FMT>(z[0], z[1], z[2], z[3]), codes4<FMT>(z[4], z[5], z[6], z[7]));
}

// largest of the 16 lanes of a row of lanes, in all of them
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false));       // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, false));
}

constexpr uint32_t kRowBlocks = 4;                   // blocks of a 16-lane team

// Blocks of 1 x 128 of x itself: 16 lanes to a block, eight elements to a lane, kRowBlocks blocks in flight.  8192 x 7168 bf16: 30.9 us, 5.8 TB/s.
// STREAM: past the caches, both ways.  From 96 MiB of x on, which the caches hold no longer than it takes to read them (8192 x 7168: 30.9 us, reading alone 32.8, neither
// 34.6); below that a product that follows finds the codes nearer.
template <int TYPE, int FMT, bool STREAM>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(const Fp8QuantArgs a) {
    constexpr uint32_t kSize = TYPE == CMX_OUT_FP32 ? 4 : 2, kTeams = 256 / 16;
    const uint32_t lane = threadIdx.x & 15u, team = threadIdx.x / 16;
    // blocks are numbered row by row; the workgroup's first one is found by a division, the others by steps from there
    const uint32_t total = a.rows * a.blocks, first = blockIdx.x * (kTeams * kRowBlocks), row0 = first / a.blocks, blk0 = first - row0 * a.blocks;
    const uint8_t* const x = a.x + blockIdx.y * a.x_step;
    float v[kRowBlocks][8];
    uint32_t row[kRowBlocks], blk[kRowBlocks];
#pragma unroll
    for (uint32_t i = 0; i < kRowBlocks; ++i) {
        const uint32_t at = blk0 + min(team + i * kTeams, total - 1 - first);
        const uint32_t down = a.blocks > kTeams * kRowBlocks ? (at >= a.blocks ? 1u : 0u) : (at * a.block_part) >> 16;      // at / a.blocks
        row[i] = row0 + down;
        blk[i] = at - down * a.blocks;
        const uint32_t col = blk[i] * kBlock + 8 * lane, n = col < a.cols ? a.cols - col : 0;
        load8<TYPE, STREAM>(x + row[i] * a.ld_x + (size_t)col * kSize, a.vec && n >= 8, n, v[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kRowBlocks; ++i) {
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, magnitude(v[i][j]));
        const BlockScale<FMT> b(max16(amax), a.pow2);
        const uint2 c = codes8<FMT>(v[i], b);
        const uint32_t col = blk[i] * kBlock + 8 * lane;
        if (first + team + i * kTeams >= total) continue;
        const size_t r = (size_t)blockIdx.y * a.rows + row[i];
        if (col < a.out_wide) {
            uint2 w = c;
            if (!b.finite && col + 8 > a.cols) {                       // the zeros behind the row stay zeros
                const uint32_t n = col < a.cols ? a.cols - col : 0;
                const uint64_t keep = n == 0 ? 0 : ~0ull >> (64 - 8 * n);
                w = make_uint2(c.x & (uint32_t)keep, c.y & (uint32_t)(keep >> 32));
            }
            v2i* const to = reinterpret_cast<v2i*>(a.codes + r * a.ld_codes + col);
            if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(v2i, w), to);
            else *to = __builtin_bit_cast(v2i, w);
        }
        if (lane == 0) a.scales[r * a.ld_scales + blk[i]] = b.s;
    }
}

// Tiles of 128 x 128 of x: blocks of 128 x 128, and both kinds of the transpose.  A thread holds 8 x 8 elements; what is turned passes through the LDS
// as codes, so that both sides of memory see whole lines.  2777 x 4096 bf16, transposed: 10.6 us, of which the launch takes 2.5 and the bytes 6.6; 8192 x 7168 45 us, in
// blocks of 128 x 128 39 (past the caches 47 and 42: these stay in them).
template <int TYPE, int FMT, bool SQUARE, bool TURNED>
__global__ __launch_bounds__(256) void fp8_quant_tile_kernel(const Fp8QuantArgs a) {
    static_assert(SQUARE || TURNED, "rows of x itself have a kernel of their own");
    constexpr uint32_t kSize = TYPE == CMX_OUT_FP32 ? 4 : 2;
    __shared__ uint32_t s_max[16][kBlock + 4];
    __shared__ float s_scale[2][kBlock];
    // row r of codes holds its 8-byte piece p at place p ^ (r / 8): the 16 threads that write pieces of rows 8 apart meet different banks
    __shared__ __attribute__((aligned(16))) uint8_t s_codes[TURNED ? kBlock * kBlock : 16];
    const uint32_t tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;      // column and row of the thread's 8 x 8
    const uint32_t col0 = blockIdx.x * kBlock, row0 = blockIdx.y * kBlock, col = col0 + 8 * tx, row = row0 + 8 * ty;
    const uint8_t* const x = a.x + blockIdx.z * a.x_step;
    const uint32_t n = col < a.cols ? a.cols - col : 0;
    float v[8][8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const bool in = row + i < a.rows && n != 0;
        if (in) {
            load8<TYPE>(x + (row + i) * a.ld_x + (size_t)col * kSize, a.vec && n >= 8, n, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        }
    }
    uint32_t most[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        most[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most[j] = max(most[j], magnitude(v[i][j]));
    }
    const size_t z0 = (size_t)blockIdx.z * a.out_rows, s0 = (size_t)blockIdx.z * a.scale_rows;
    if constexpr (SQUARE) {
        uint32_t all = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) all = max(all, most[j]);
        all = max16(all);
        if (tx == 0) s_max[0][ty] = all;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) all = max(all, s_max[0][i]);
        const BlockScale<FMT> b(all, a.pow2);
        if (threadIdx.x == 0) a.scales[(s0 + (TURNED ? blockIdx.x : blockIdx.y)) * a.ld_scales + (TURNED ? blockIdx.y : blockIdx.x)] = b.s;
        if constexpr (!TURNED) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                uint2 w = codes8<FMT>(v[i], b);
                if (row + i >= a.rows || col >= a.out_wide) continue;
                if (!b.finite && n < 8) {
                    const uint64_t keep = n == 0 ? 0 : ~0ull >> (64 - 8 * n);
                    w = make_uint2(w.x & (uint32_t)keep, w.y & (uint32_t)(keep >> 32));
                }
                *reinterpret_cast<uint2*>(a.codes + (z0 + row + i) * a.ld_codes + col) = w;
            }
            return;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                float t[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = v[i][j];
                *reinterpret_cast<uint2*>(s_codes + (8 * tx + j) * kBlock + 8 * (ty ^ tx)) = codes8<FMT>(t, b);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) s_max[ty][8 * tx + j] = most[j];
        __syncthreads();
        if (threadIdx.x < kBlock) {                                    // a thread to a column
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, s_max[i][threadIdx.x]);
            const BlockScale<FMT> b(m, a.pow2);
            s_scale[0][threadIdx.x] = b.s;
            s_scale[1][threadIdx.x] = b.inverse;
            if (col0 + threadIdx.x < a.cols) a.scales[(s0 + col0 + threadIdx.x) * a.ld_scales + blockIdx.y] = b.s;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const float scale = s_scale[0][8 * tx + j];
            const BlockScale<FMT> b(scale, s_scale[1][8 * tx + j], magnitude(scale) < kInfBits);
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = v[i][j];
            *reinterpret_cast<uint2*>(s_codes + (8 * tx + j) * kBlock + 8 * (ty ^ tx)) = codes8<FMT>(t, b);
        }
    }
    if constexpr (TURNED) {
        __syncthreads();
        // out rows are columns of x; eight lanes to a row, 16 bytes each
        const uint32_t piece = threadIdx.x & 7u, out_col = row0 + 16 * piece;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t r = threadIdx.x / 8 + 32 * i;
            if (col0 + r >= a.cols || out_col >= a.out_wide) continue;
            uint64_t w[2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) w[h] = *reinterpret_cast<const uint64_t*>(s_codes + r * kBlock + 8 * ((2 * piece + h) ^ (r >> 3)));
            const uint32_t left = a.out_cols > out_col ? a.out_cols - out_col : 0;       // (behind them zeros, also in a block that is not finite)
            if (left < 16) {
                w[1] = left <= 8 ? 0 : w[1] & (~0ull >> (128 - 8 * left));
                if (left < 8) w[0] = left == 0 ? 0 : w[0] & (~0ull >> (64 - 8 * left));
            }
            *reinterpret_cast<uint4*>(a.codes + (z0 + col0 + r) * a.ld_codes + out_col) =
                make_uint4((uint32_t)w[0], (uint32_t)(w[0] >> 32), (uint32_t)w[1], (uint32_t)(w[1] >> 32));
        }
    }
}

template <int TYPE, int FMT>
int launch(const Fp8QuantArgs& a, uint32_t batch, bool square, bool turned, hipStream_t s) {
    if (!square && !turned) {
        const uint64_t groups = ((uint64_t)a.rows * a.blocks + 16 * kRowBlocks - 1) / (16 * kRowBlocks);
        CMX_REQUIRE((uint64_t)a.rows * a.blocks < (1ull << 31) && fits_grid(groups, 256), "too many elements");
        const bool stream = (uint64_t)batch * a.rows * a.cols * (TYPE == CMX_OUT_FP32 ? 4 : 2) >= 96ull << 20;
        hipLaunchKernelGGL((stream ? fp8_quant_rows_kernel<TYPE, FMT, true> : fp8_quant_rows_kernel<TYPE, FMT, false>), dim3((uint32_t)groups, batch), dim3(256), 0, s, a);
    } else {
        const uint32_t bx = ceil_div(a.cols, kBlock), by = ceil_div(a.rows, kBlock);
        CMX_REQUIRE(by <= 65535u && fits_grid(bx, 256), "too many rows or columns");
        const auto kfn = square ? (turned ? fp8_quant_tile_kernel<TYPE, FMT, true, true> : fp8_quant_tile_kernel<TYPE, FMT, true, false>)
                                : fp8_quant_tile_kernel<TYPE, FMT, false, true>;
        hipLaunchKernelGGL(kfn, dim3(bx, by, batch), dim3(256), 0, s, a);
    }
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

template <int TYPE>
int launch(const Fp8QuantArgs& a, uint32_t batch, int fmt, bool square, bool turned, hipStream_t s) {
    return fmt == CMX_FMT_E5M2 ? launch<TYPE, CMX_FMT_E5M2>(a, batch, square, turned, s) : launch<TYPE, CMX_FMT_E4M3>(a, batch, square, turned, s);
}

}  // namespace
}  // namespace cmx

int cmx::preload_fp8_quant_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::fp8_quant_rows_kernel<CMX_OUT_BF16, CMX_FMT_E4M3, false>)));
    return CMX_OK;
}

extern "C" int cmx_fp8_block_quant(const void* x, uint32_t ld_x, uint64_t x_step, int type, uint8_t* codes, uint32_t ld_codes, float* scales,
                                   uint32_t ld_scales, uint32_t batch, uint32_t rows, uint32_t cols, int fmt, int square, int transposed, int pow2,
                                   cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(type == CMX_OUT_BF16 || type == CMX_OUT_FP16 || type == CMX_OUT_FP32, "unknown type");
    CMX_REQUIRE(fmt == CMX_FMT_E4M3 || fmt == CMX_FMT_E5M2, "8-bit formats only");
    if (batch == 0 || rows == 0 || cols == 0) return CMX_OK;
    CMX_REQUIRE(x && codes && scales, "null pointer");
    CMX_REQUIRE(rows < (1u << 31) && cols < (1u << 31), "at most 2^31 - 1 rows and columns");
    CMX_REQUIRE(batch <= 65535u, "at most 65535 matrices");
    const uint32_t size = type == CMX_OUT_FP32 ? 4 : 2;
    const uint32_t out_rows = transposed ? cols : rows, out_cols = transposed ? rows : cols;
    const uint32_t wide = round_up(out_cols, 16), blocks = ceil_div(out_cols, kBlock), scale_rows = square ? ceil_div(out_rows, kBlock) : out_rows;
    CMX_REQUIRE(ld_x >= cols && ld_codes >= wide && ld_scales >= blocks, "row pitch smaller than row");
    CMX_REQUIRE(reinterpret_cast<uintptr_t>(x) % size == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0, "pointers must be aligned to their elements");
    CMX_REQUIRE(aligned16(codes) && ld_codes % 16 == 0, "rows of codes must be 16-byte aligned");
    Fp8QuantArgs a = {static_cast<const uint8_t*>(x), codes, scales, (size_t)ld_x * size, (size_t)x_step * size, ld_codes, ld_scales, rows, cols,
                      out_cols, wide, out_rows, scale_rows, blocks, 0, pow2 ? 1u : 0u, 65535u / blocks + 1};
    a.vec = aligned16(x) && a.ld_x % 16 == 0 && (batch == 1 || a.x_step % 16 == 0) ? 1u : 0u;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == CMX_OUT_BF16) return launch<CMX_OUT_BF16>(a, batch, fmt, square != 0, transposed != 0, s);
    return type == CMX_OUT_FP16 ? launch<CMX_OUT_FP16>(a, batch, fmt, square != 0, transposed != 0, s)
                                : launch<CMX_OUT_FP32>(a, batch, fmt, square != 0, transposed != 0, s);
}
