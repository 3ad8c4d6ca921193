// Residual addition, root-mean-square norm and MX quantisation in one pass over the rows.
//
//   t = x + residual,   r = 1 / sqrt(mean(t^2) + eps),   y = t * r * weight
//
// in fp32; t and y are rounded once each, to the type of x, and codes and scales are those of the exact y of t (finish8).  A row is read
// once: its elements stay in registers between the sum of squares and the scaling (a row that is too long for the registers of one
// workgroup is read twice, the second time mostly from the caches).
// Work split: a thread holds pieces of eight consecutive elements, so that four neighbouring lanes hold one MX block, whose
// maximum is then two DPP exchanges away.  Short rows are a wavefront's, which needs no barrier, longer ones a workgroup's.
// Bound by memory.  bf16 rows with a residual and total: 8192 x 7168 to E4M3 codes in 80 us (5.2 TB/s, as a plain copy; E2M1 76), to bf16 in 83 (5.6 TB/s), of
// 4096 columns to bf16 5.6 to 5.9 TB/s; rows of odd length, whose pieces lie across cache lines, 3.5 to 4.3.  A single row takes 3.2 us, of which 2.5 are the launch's.
#include "mx_launch.h"

namespace cmx {
namespace {

constexpr int kBf16 = CMX_OUT_BF16, kFp16 = CMX_OUT_FP16, kFp32 = CMX_OUT_FP32;

template <int TYPE>
struct Elem {
    static constexpr uint32_t bytes = TYPE == kFp32 ? 4 : 2;
};

// Eight elements as they lie in memory.  Rows need only the alignment of an element: global loads and stores of 16 bytes may lie at any address.
template <int TYPE>
struct Raw {
    uint32_t w[TYPE == kFp32 ? 8 : 4];
};

template <int TYPE>
__device__ __forceinline__ float value(const Raw<TYPE>& r, int i) {
    if constexpr (TYPE == kFp32) return __uint_as_float(r.w[i]);
    const uint32_t bits = (i & 1) ? r.w[i >> 1] >> 16 : r.w[i >> 1] & 0xFFFFu;
    if constexpr (TYPE == kBf16) return bf16_to_f32(bits);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// a whole piece at p, or zeros
template <int TYPE>
__device__ __forceinline__ Raw<TYPE> load8(const uint8_t* p, bool whole) {
    Raw<TYPE> r;
#pragma unroll
    for (uint32_t i = 0; i < sizeof(r) / 4; ++i) r.w[i] = 0;
    if (whole) __builtin_memcpy(&r, p, sizeof(r));
    return r;
}

// the first left < 8 elements at p, into a piece of zeros: the end of a row.  Apart from load8, so that the loads of all whole
// pieces are under way before anything waits for these.
template <int TYPE>
__device__ __forceinline__ void load_end(Raw<TYPE>& r, const uint8_t* p, uint32_t left) {
#pragma unroll
    for (uint32_t i = 0; i < 7; ++i) {
        if (i >= left) continue;
        if constexpr (TYPE == kFp32) {
            r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
            r.w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
        }
    }
}

// v rounded to TYPE, to the first `left` elements at p
template <int TYPE>
__device__ __forceinline__ void store8(uint8_t* p, const float (&v)[8], uint32_t left) {
    Raw<TYPE> r;
    if constexpr (TYPE == kFp32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(v[i]);
    } else if constexpr (TYPE == kBf16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = cvt_pk_bf16(v[2 * i], v[2 * i + 1]);
    } else {
        typedef _Float16 v2f16 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = __builtin_bit_cast(uint32_t, (v2f16){(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
    }
    if (left >= 8) {
        __builtin_memcpy(p, &r, sizeof(r));
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        if (i >= left) continue;
        if constexpr (TYPE == kFp32) {
            reinterpret_cast<uint32_t*>(p)[i] = r.w[i];
        } else {
            reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(r.w[i >> 1] >> (16 * (i & 1)));
        }
    }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
}

// Eight codes of y under the scale of its block (four lanes), nearest even, by the rules of cmx_mx_quant: shared exponent from the block's
// maximum, magnitudes above the largest code clipped, Inf to the largest code, NaN to the NaN code (4 bits: scale 255, codes zero).
// Returns the scale byte.
template <int FMT>
__device__ __forceinline__ uint32_t quantize8(const float (&y)[8], uint32_t (&w)[2]) {
    constexpr bool kFp4 = FMT == CMX_FMT_E2M1;
    constexpr int emax = FMT == CMX_FMT_E4M3 ? kEmaxE4M3 : (FMT == CMX_FMT_E5M2 ? kEmaxE5M2 : kEmaxE2M1);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    amax = quad_max(amax);
    const bool nonfinite = amax >= 0x7F800000u;
    int e = (int)(amax >> 23) - 127 - emax;
    if (kFp4 && nonfinite) e = 127;
    e = amax < __float_as_uint(1e-12f) ? 0 : e;
    // the largest code's value under this scale: the block's own exponent with the mantissa of 448, 57344 (1.75) or 6 (1.5)
    const float lim = nonfinite ? 3.402823466e38f : __uint_as_float(((uint32_t)(e + emax + 127) << 23) | (kFp4 ? 0x400000u : 0x600000u));
    const float scale = __uint_as_float((uint32_t)(e + 127) << 23);
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_fmed3f(y[i], -lim, lim);
    w[0] = w[1] = 0;
    if constexpr (kFp4) {
        w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], c[0], c[1], scale, 0);
        w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], c[2], c[3], scale, 1);
        w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], c[4], c[5], scale, 2);
        w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], c[6], c[7], scale, 3);
        if (nonfinite) {
            // scale 2^127: 2^127 itself is code 1.0 and nothing finite reaches 2.0; Inf the largest code, a NaN in the block clears it
            w[0] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[0] |= e2m1_encode(clamp_abs(ldexpf(y[i], -127), 6.0f), false) << (4 * i);
            if (amax > 0x7F800000u) w[0] = 0;
        }
        return amax > 0x7F800000u ? 255u : (uint32_t)(e + 127);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v2i16 o = {0, 0};
            if constexpr (FMT == CMX_FMT_E4M3) {
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, c[4 * h], c[4 * h + 1], scale, false);
                o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, c[4 * h + 2], c[4 * h + 3], scale, true);
            } else {
                o = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(o, c[4 * h], c[4 * h + 1], scale, false);
                o = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(o, c[4 * h + 2], c[4 * h + 3], scale, true);
            }
            w[h] = __builtin_bit_cast(uint32_t, o);
        }
        if (nonfinite) {
            constexpr uint32_t maxc = FMT == CMX_FMT_E5M2 ? 0x7Bu : 0x7Eu;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t bits = __float_as_uint(y[i]), mag = bits & 0x7FFFFFFFu, sign = (bits >> 24) & 0x80u, sh = 8 * (i & 3);
                if (mag >= 0x7F800000u) w[i >> 2] = (w[i >> 2] & ~(0xFFu << sh)) | ((mag == 0x7F800000u ? maxc | sign : 0x7Fu | sign) << sh);
            }
        }
        return (uint32_t)(e + 127);
    }
}

// d to fp32 so that a later rounding to fewer bits, and the exponent, are those of d: towards zero, the last bit set if anything was cut off
__device__ __forceinline__ float to_odd(double d) {
    const float f = (float)d;
    uint32_t bits = __float_as_uint(f);
    if (fabs((double)f) > fabs(d)) --bits;
    if ((double)f != d) bits |= 1u;
    return __uint_as_float(bits);
}

struct NormArgs {
    const uint8_t* x;
    const uint8_t* residual;   // may be null
    const uint8_t* weight;
    uint8_t* total;            // may be null; may be x or residual: an element is read before it is written, by the same thread
    uint8_t* y;                // may be null
    uint8_t* codes;            // may be null
    uint8_t* scales;
    size_t ld_x, ld_residual, ld_total, ld_y, ld_codes, ld_scales;      // bytes
    uint32_t rows, cols;
    float eps;
    int fmt;
};

// where a piece's results go; v = t, the weight beside it; every lane of a quad comes here
// squares: the sum over the row, rstd from it in fp32
template <int TYPE, int WTYPE>
__device__ __forceinline__ void finish8(const NormArgs& a, size_t row, uint32_t col, const float (&v)[8], const Raw<WTYPE>& weight, float rstd, double squares, float eps) {
    const uint32_t left = col < a.cols ? a.cols - col : 0;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (uint32_t)i < left ? v[i] * rstd * value<WTYPE>(weight, i) : 0.0f;
    if (a.y && left) store8<TYPE>(a.y + row * a.ld_y + (size_t)col * Elem<TYPE>::bytes, y, left);
    if (!a.codes) return;
    // Codes and scale are to be those of the exact y.  In fp32 it is off by less than kNear units in the last place, which matters next to a border between
    // codes or a power of two: places where the bits that no code keeps are zeros (a border's last bit is one behind a code's).  There, in one piece of
    // 60, the wavefront computes its y again in 64 bits.  (8192 x 7168 bf16, residual: 80 us, without this 76 and 36 of 59 million codes on the wrong side.)
    constexpr uint32_t kNear = 8;
    const uint32_t kept = a.fmt == CMX_FMT_E4M3 ? 13 : (a.fmt == CMX_FMT_E5M2 ? 12 : 11);
    const auto place = [&](float f) { return (__float_as_uint(f) << kept) + (kNear << kept); };
    uint32_t nearest = ~0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) nearest = min(nearest, place(y[i]));
    if (__any(nearest <= 2 * kNear << kept)) {
        bool near = false;                                                   // (zeros are near by their bits only)
#pragma unroll
        for (int i = 0; i < 8; ++i) near |= y[i] != 0.0f && place(y[i]) <= 2 * kNear << kept;
        if (__any(near) && rstd > 0.0f) {                                    // (0: the squares passed fp32)
            asm volatile("" : "+v"(squares));                                // (or what this needs is computed, or held in 64 bits, by all)
            const double exact = 1.0 / sqrt(squares / (double)a.cols + (double)eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float t = v[i];
                asm volatile("" : "+v"(t));
                y[i] = (uint32_t)i < left ? to_odd((double)t * exact * (double)value<WTYPE>(weight, i)) : 0.0f;
            }
        }
    }
    uint32_t w[2], byte;
    if (a.fmt == CMX_FMT_E4M3) byte = quantize8<CMX_FMT_E4M3>(y, w);
    else if (a.fmt == CMX_FMT_E5M2) byte = quantize8<CMX_FMT_E5M2>(y, w);
    else byte = quantize8<CMX_FMT_E2M1>(y, w);
    if (!left) return;
    if (a.fmt == CMX_FMT_E2M1) {
        uint8_t* o = a.codes + row * a.ld_codes + (col >> 1);
        if (left >= 8) {
            __builtin_memcpy(o, w, 4);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (2 * i < left) o[i] = (uint8_t)(w[0] >> (8 * i));
        }
    } else {
        uint8_t* o = a.codes + row * a.ld_codes + col;
        if (left >= 8) {
            __builtin_memcpy(o, w, 8);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (i < left) o[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
        }
    }
    if ((col & 31u) == 0) {
        uint8_t* s = a.scales + row * a.ld_scales;
        const uint32_t kb = col >> 5, nb = (a.cols + 31) >> 5;
        s[kb] = (uint8_t)byte;
        if (kb == nb - 1 && (nb & 1u) && a.ld_scales > nb) s[nb] = 127;      // pad the scale row to an even count with 1.0
    }
}

// sum over the TPR threads of a row; every one of them gets it
template <int TPR>
__device__ __forceinline__ double row_sum(double v, double* shared) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += shared[i];
    }
    return v;
}

__device__ __forceinline__ float inverse_rms(float squares, uint32_t cols, float eps) { return 1.0f / sqrtf(squares / (float)cols + eps); }

// Rows whose squares fp32 holds in part or not at all, beside an eps that is as small or zero: t is lifted by a power of two, squares and eps by its square, which
// leaves y as it is.  From the smallest t on (2^-149) the mean of up to 2^30 squares is then a normal number, and none is too large.
constexpr float kLift = 0x1p104f;
__device__ __forceinline__ bool needs_lift(double squares, float eps) { return squares < 0x1p-90 && eps < 0x1p-90f; }

// TPR threads per row, PIECES pieces of eight elements per thread: rows of up to 8 * TPR * PIECES elements
template <int TYPE, int WTYPE, int TPR, int PIECES>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_kernel(const NormArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR;
    __shared__ double shared[kThreads / 64];
    const uint32_t lane = threadIdx.x % TPR;
    const size_t row = (size_t)blockIdx.x * kRows + threadIdx.x / TPR;
    if (kRows > 1 && row >= a.rows) return;                                  // (whole wavefronts; such rows share no barrier)
    float v[PIECES][8];
    Raw<TYPE> x[PIECES], r[PIECES];
    Raw<WTYPE> w[PIECES];
    const uint8_t *const xr = a.x + row * a.ld_x, *const rr = a.residual + row * a.ld_residual;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const uint32_t col = (lane + p * TPR) * 8;
        const bool whole = col + 8 <= a.cols;
        x[p] = load8<TYPE>(xr + (size_t)col * Elem<TYPE>::bytes, whole);
        if (a.residual) r[p] = load8<TYPE>(rr + (size_t)col * Elem<TYPE>::bytes, whole);
        w[p] = load8<WTYPE>(a.weight + (size_t)col * Elem<WTYPE>::bytes, whole);
    }
    if (a.cols & 7u) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t col = (lane + p * TPR) * 8, left = a.cols & 7u;
            if (col != a.cols - left) continue;
            load_end<TYPE>(x[p], xr + (size_t)col * Elem<TYPE>::bytes, left);
            if (a.residual) load_end<TYPE>(r[p], rr + (size_t)col * Elem<TYPE>::bytes, left);
            load_end<WTYPE>(w[p], a.weight + (size_t)col * Elem<WTYPE>::bytes, left);
        }
    }
    double squares = 0.0;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const uint32_t col = (lane + p * TPR) * 8, left = col < a.cols ? a.cols - col : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[p][i] = value<TYPE>(x[p], i) + (a.residual ? value<TYPE>(r[p], i) : 0.0f);
            squares = fma((double)v[p][i], (double)v[p][i], squares);
        }
        if (a.total && left) store8<TYPE>(a.total + row * a.ld_total + (size_t)col * Elem<TYPE>::bytes, v[p], left);
    }
    squares = row_sum<TPR>(squares, shared);
    float eps = a.eps;
    if (needs_lift(squares, eps)) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] *= kLift;
        }
        squares *= (double)kLift * kLift;
        eps = eps * kLift * kLift;
    }
    const float rstd = inverse_rms((float)squares, a.cols, eps);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const uint32_t col = (lane + p * TPR) * 8;
        if (col - (lane & 3) * 8 < a.cols) finish8<TYPE, WTYPE>(a, row, col, v[p], w[p], rstd, squares, eps);      // (whole quads)
    }
}

// rows of any length: two passes
template <int TYPE, int WTYPE>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(const NormArgs a) {
    __shared__ double shared[16];
    const size_t row = blockIdx.x;
    // elements [col, col + 8) of t, zeros behind the row
    const auto piece = [&](uint32_t col, float (&v)[8]) {
        const bool whole = col + 8 <= a.cols;
        const uint8_t *const xp = a.x + row * a.ld_x + (size_t)col * Elem<TYPE>::bytes,
                      *const rp = a.residual + row * a.ld_residual + (size_t)col * Elem<TYPE>::bytes;
        Raw<TYPE> x = load8<TYPE>(xp, whole), r;
        if (a.residual) r = load8<TYPE>(rp, whole);
        if (!whole && col < a.cols) {
            load_end<TYPE>(x, xp, a.cols - col);
            if (a.residual) load_end<TYPE>(r, rp, a.cols - col);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = value<TYPE>(x, i) + (a.residual ? value<TYPE>(r, i) : 0.0f);
    };
    double squares = 0.0;
    float v[8];
    for (uint32_t col = threadIdx.x * 8; col < a.cols; col += 8192) {
        piece(col, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) squares = fma((double)v[i], (double)v[i], squares);
    }
    squares = row_sum<1024>(squares, shared);
    float eps = a.eps;
    const bool lift = needs_lift(squares, eps);
    if (lift) {
        squares *= (double)kLift * kLift;
        eps = eps * kLift * kLift;
    }
    const float rstd = inverse_rms((float)squares, a.cols, eps);
    for (uint32_t col = threadIdx.x * 8; col - (threadIdx.x & 3) * 8 < a.cols; col += 8192) {        // (whole quads)
        piece(col, v);
        const uint8_t* const wp = a.weight + (size_t)col * Elem<WTYPE>::bytes;
        Raw<WTYPE> w = load8<WTYPE>(wp, col + 8 <= a.cols);
        if (col < a.cols && col + 8 > a.cols) load_end<WTYPE>(w, wp, a.cols - col);
        if (a.total && col < a.cols) store8<TYPE>(a.total + row * a.ld_total + (size_t)col * Elem<TYPE>::bytes, v, a.cols - col);
        if (lift) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= kLift;
        }
        finish8<TYPE, WTYPE>(a, row, col, v, w, rstd, squares, eps);
    }
}

template <int TYPE, int WTYPE>
int launch(const NormArgs& a, hipStream_t s) {
    const auto run = [&](auto kernel, uint32_t rows_each, uint32_t threads) {
        hipLaunchKernelGGL(kernel, dim3(ceil_div(a.rows, rows_each)), dim3(threads), 0, s, a);
        CMX_LAUNCH_CHECK();
        return CMX_OK;
    };
    if (a.cols <= 512) return run(rms_norm_kernel<TYPE, WTYPE, 64, 1>, 4, 256);
    if (a.cols <= 1024) return run(rms_norm_kernel<TYPE, WTYPE, 64, 2>, 4, 256);
    if (a.cols <= 2048) {
        // A wavefront or a workgroup to a row of 16 bits: the former waits for nobody, the latter has shorter rows.  us with codes, 1348 columns: 1024 rows 8.8
        // and 7.9, 5041 rows 15.6 and 18.6, 32768 rows 77 and 103; 2048 columns, 32768 rows 88 and 93 (of 32 bits 169 and 158).
        if constexpr (TYPE != kFp32) {
            int cus;
            if (int rc = cu_count(&cus); rc != CMX_OK) return rc;
            if (a.rows >= 16u * (uint32_t)cus) return run(rms_norm_kernel<TYPE, WTYPE, 64, 4>, 4, 256);
        }
        return run(rms_norm_kernel<TYPE, WTYPE, 256, 1>, 1, 256);
    }
    if (a.cols <= 4096) return run(rms_norm_kernel<TYPE, WTYPE, 256, 2>, 1, 256);
    if (a.cols <= 8192) return run(rms_norm_kernel<TYPE, WTYPE, 256, 4>, 1, 256);
    if (a.cols <= 16384) return run(rms_norm_kernel<TYPE, WTYPE, 1024, 2>, 1, 1024);
    return run(rms_norm_long_kernel<TYPE, WTYPE>, 1, 1024);
}

}  // namespace
}  // namespace cmx

int cmx::preload_norm_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::rms_norm_long_kernel<CMX_OUT_BF16, CMX_OUT_BF16>)));
    return CMX_OK;
}

extern "C" int cmx_rms_norm_quant(const void* x, uint32_t ld_x, const void* residual, uint32_t ld_residual, const void* weight,
                                  void* total, uint32_t ld_total, void* y, uint32_t ld_y, uint8_t* codes, uint32_t ld_codes,
                                  uint8_t* scales, uint32_t ld_scales, uint32_t rows, uint32_t cols, uint32_t eps_bits, int type,
                                  int weight_type, int fmt, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(type == kBf16 || type == kFp16 || type == kFp32, "unknown type");
    CMX_REQUIRE(weight_type == type || weight_type == kFp32, "the weight must be of the type of x or fp32");
    CMX_REQUIRE(!codes || fmt == CMX_FMT_E4M3 || fmt == CMX_FMT_E5M2 || fmt == CMX_FMT_E2M1, "unknown element format");
    float eps;
    __builtin_memcpy(&eps, &eps_bits, 4);
    CMX_REQUIRE(eps >= 0.0f && eps < 3.402823466e38f, "eps must be a finite number, not negative");
    if (rows == 0 || cols == 0) return CMX_OK;
    CMX_REQUIRE(x && weight, "null pointer");
    CMX_REQUIRE(y || codes, "nothing to write: y or codes");
    CMX_REQUIRE((codes != nullptr) == (scales != nullptr), "codes and scales come together");
    CMX_REQUIRE(!total || residual, "a total needs a residual");
    const uint32_t bytes = type == kFp32 ? 4 : 2, nb = ceil_div(cols, 32);
    CMX_REQUIRE(ld_x >= cols && (!residual || ld_residual >= cols) && (!total || ld_total >= cols) && (!y || ld_y >= cols), "row pitch smaller than row");
    CMX_REQUIRE(!codes || (ld_codes >= (fmt == CMX_FMT_E2M1 ? ceil_div(cols, 2) : cols) && (ld_scales == nb || ld_scales >= scale_cols(cols))),
                "row pitch smaller than row");
    const auto off = [](const void* p, uint32_t by) { return reinterpret_cast<uintptr_t>(p) % by != 0; };
    CMX_REQUIRE(!off(x, bytes) && !off(residual, bytes) && !off(total, bytes) && !off(y, bytes) && !off(weight, weight_type == kFp32 ? 4 : 2),
                "pointers must be aligned to their elements");
    CMX_REQUIRE(cols <= (1u << 30), "row too long");
    CMX_REQUIRE(fits_grid((uint64_t)rows + 3, cols <= 1024 ? 64 : (cols <= 8192 ? 256 : 1024)), "too many rows");      // (+ 3: a workgroup of four rows)
    const NormArgs a = {static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(residual), static_cast<const uint8_t*>(weight),
                        static_cast<uint8_t*>(total), static_cast<uint8_t*>(y), codes, scales, (size_t)ld_x * bytes, (size_t)ld_residual * bytes,
                        (size_t)ld_total * bytes, (size_t)ld_y * bytes, ld_codes, ld_scales, rows, cols, eps, fmt};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == kBf16) return weight_type == kBf16 ? launch<kBf16, kBf16>(a, s) : launch<kBf16, kFp32>(a, s);
    if (type == kFp16) return weight_type == kFp16 ? launch<kFp16, kFp16>(a, s) : launch<kFp16, kFp32>(a, s);
    return launch<kFp32, kFp32>(a, s);
}
