// A few rows of 16- or 32-bit activations times MXFP4 weights: the tile of one wavefront.
//
// The weights are the matrix instruction's rows: v_mfma_f32_16x16x32_bf16 takes 16 weight rows and up to 16 activation rows as its
// columns.  E2M1 times a power of two is exact in bf16 and an activation is one bf16 value or a sum of two or three (fp16, fp32), so
// every product is exact and sums are fp32: nothing is rounded before the result.  Which K a lane's eight values stand for is free as long as
// both operands agree, so that a lane's share of a step is what it loads at once: 16 bytes of its weight row = 32 codes = one block with
// one scale, feeding four instructions.  Lane l: row (or column) l % 16, block l / 16 of the step's four.
#pragma once

#include "mx_common.h"

namespace cmx {

typedef __bf16 v8bf16 __attribute__((ext_vector_type(8)));

constexpr uint32_t kStepK = 128;         // K of one step: four blocks, one for each 16 lanes

// ---- activations ----------------------------------------------------------------------------------------------------
enum XKind { kXBf16 = CMX_OUT_BF16, kXFp16 = CMX_OUT_FP16, kXFp32 = CMX_OUT_FP32, kXPlanes = 3 };

// 32 consecutive activations of one row, as loaded.  kXPlanes: two bf16 arrays, `plane` bytes apart, whose sum is the value.
template <int KIND>
struct XRegs {
    static constexpr int kLoads = KIND == kXFp32 || KIND == kXPlanes ? 8 : 4;
    static constexpr int kPieces = KIND == kXBf16 ? 1 : (KIND == kXFp32 ? 3 : 2);
    static constexpr uint32_t kBytes = KIND == kXFp32 ? 4 : 2;      // of an element, in one array
    uint4 r[kLoads];

    __device__ __forceinline__ void load(const uint8_t* p, size_t plane) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) __builtin_memcpy(&r[i], KIND == kXPlanes && i >= 4 ? p + plane + 16 * (i - 4) : p + 16 * i, 16);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) r[i] = make_uint4(0, 0, 0, 0);
    }
    // values [8 j, 8 j + 8) as kPieces operands; a value is the sum of its pieces, exactly: each takes the leading eight bits of what is left
    __device__ __forceinline__ void pieces(int j, v8bf16 (&out)[kPieces]) const {
        if constexpr (KIND == kXBf16) {
            out[0] = __builtin_bit_cast(v8bf16, r[j]);
        } else if constexpr (KIND == kXPlanes) {
            out[0] = __builtin_bit_cast(v8bf16, r[j]);
            out[1] = __builtin_bit_cast(v8bf16, r[4 + j]);
        } else {
            float v[8];
            if constexpr (KIND == kXFp16) {
                typedef _Float16 v8f16 __attribute__((ext_vector_type(8)));
                const v8f16 h = __builtin_bit_cast(v8f16, r[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
            } else {
                const uint4 a = r[2 * j], b = r[2 * j + 1];
                const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
            }
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = __builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);      // upper halves
                out[p] = __builtin_bit_cast(v8bf16, make_uint4(w[0], w[1], w[2], w[3]));
                if (p + 1 < kPieces) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float lead = __uint_as_float(__float_as_uint(v[i]) & 0xFFFF0000u);
                        v[i] = lead == v[i] ? 0.0f : v[i] - lead;          // (Inf leaves nothing, a NaN a NaN)
                    }
                }
            }
        }
    }
};

// ---- weights --------------------------------------------------------------------------------------------------------
// E8M0 byte -> the float that scales a conversion: 2^(byte - 127), NaN for 255
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    const uint32_t bits = byte == 0 ? 0x00400000u : byte << 23;
    return __uint_as_float(byte == 255 ? 0x7FC00000u : bits);
}

// eight E2M1 codes times a scale
__device__ __forceinline__ v8bf16 e2m1_to_bf16(uint32_t codes, float scale) {
    uint4 w;
    w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    w.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    w.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    return __builtin_bit_cast(v8bf16, w);
}

// ---- the tile -------------------------------------------------------------------------------------------------------
// RT x 16 weight rows times CT x 16 activation rows over units [first, last) of UNIT steps, every `by`-th.  The pointers are a lane's own: weight row
// (l % 16) of each row tile at its first step's block l / 16, scales likewise, activation row l % 16 of each column tile at that block.
// blocks: K / 32.
template <int KIND, int RT, int CT, int UNIT>
struct RowsTile {
    const uint8_t *a[RT], *scale[RT], *x[CT];
    size_t plane;
    uint32_t blocks;
    v4f acc[RT][CT];

    struct Regs {
        uint4 a[UNIT][RT];
        uint32_t scale[UNIT][RT];
        XRegs<KIND> x[UNIT][CT];
    };

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < CT; ++j) acc[i][j] = (v4f){0, 0, 0, 0};
    }
    __device__ __forceinline__ void load(Regs& g, uint32_t unit) const {
        const uint32_t q = (threadIdx.x & 63) >> 4;
        const bool whole = (unit + 1) * UNIT * 4 <= blocks;                 // the same for every lane
#pragma unroll
        for (int s = 0; s < UNIT; ++s) {
            const uint32_t step = unit * UNIT + s;
            const bool live = whole || step * 4 + q < blocks;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (live) {
                    g.a[s][i] = *reinterpret_cast<const uint4*>(a[i] + (size_t)step * (kStepK / 2));
                    g.scale[s][i] = scale[i][step * 4];
                } else {
                    g.a[s][i] = make_uint4(0, 0, 0, 0);
                    g.scale[s][i] = 127;
                }
            }
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                if (live) g.x[s][j].load(x[j] + (size_t)step * kStepK * XRegs<KIND>::kBytes, plane);
                else g.x[s][j].clear();
            }
        }
    }
    __device__ __forceinline__ void multiply(const Regs& g) {
#pragma unroll
        for (int s = 0; s < UNIT; ++s) {
            float f[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) f[i] = e8m0_value(g.scale[s][i]);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                v8bf16 xs[CT][XRegs<KIND>::kPieces];
#pragma unroll
                for (int j = 0; j < CT; ++j) g.x[s][j].pieces(h, xs[j]);
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const uint4 codes = g.a[s][i];
                    const v8bf16 w = e2m1_to_bf16(h == 0 ? codes.x : (h == 1 ? codes.y : (h == 2 ? codes.z : codes.w)), f[i]);
#pragma unroll
                    for (int j = 0; j < CT; ++j)
#pragma unroll
                        for (int p = 0; p < XRegs<KIND>::kPieces; ++p) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, xs[j][p], acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    // the loads of a unit are under way while the one before it is multiplied
    __device__ __forceinline__ void run(uint32_t first, uint32_t last, uint32_t by) {
        if (first >= last) return;
        Regs now;
        load(now, first);
        for (uint32_t u = first + by; u < last; u += by) {
            Regs next;
            load(next, u);
            multiply(now);
            now = next;
        }
        multiply(now);
    }
};

}  // namespace cmx
