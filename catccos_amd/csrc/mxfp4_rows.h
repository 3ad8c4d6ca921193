// A few rows of 16- or 32-bit activations times MXFP4 weights: the work of one wavefront.
//
// The weights are the matrix instruction's rows: v_mfma_f32_16x16x32_bf16 takes 16 weight rows and up to 16 activation rows as its
// columns.  E2M1 times a power of two is exact in bf16 and an activation is one bf16 value or a sum of two or three (fp16, fp32), so
// every product is exact and sums are fp32: nothing is rounded before the result.  Which K a lane's eight values stand for is free as long as
// both operands agree, so that a lane's share of a step is what it loads at once: 16 bytes of its weight row = 32 codes = one block with
// one scale, feeding four instructions.  Lane l: row (or column) l % 16, block l / 16 of the step's four.
//
// What bounds this is the vector memory path of a CU, not the matrix or vector units.  Reading weights in this layout, 1168384 rows of 1024 bytes
// (1.2 GB, cold): 6.6 TB/s alone; 5.0 with a byte of scales per lane and step; 6.5 with four bytes per lane and four steps; 3.9 with four
// loads a step for a single activation row, 1.8 with 16 rows.  So scales come as one word per unit of four steps and change lanes in
// registers, and activations come as whole kilobytes straight to LDS, from where a step reads its operands.
#pragma once

#include "mx_common.h"

namespace cmx {

typedef __bf16 v8bf16 __attribute__((ext_vector_type(8)));

constexpr uint32_t kUnitSteps = 4, kUnitBlocks = 16, kUnitK = 512;        // a step: four blocks of 32 along K, one for each 16 lanes

// ---- activations ----------------------------------------------------------------------------------------------------
// kXPlanes: two bf16 arrays, `plane` bytes apart, whose sum is the value
enum XKind { kXBf16 = CMX_OUT_BF16, kXFp16 = CMX_OUT_FP16, kXFp32 = CMX_OUT_FP32, kXPlanes = 3 };

template <int KIND>
struct XTraits {
    static constexpr int kPieces = KIND == kXBf16 ? 1 : (KIND == kXFp32 ? 3 : 2);
    static constexpr int kLoads = KIND == kXFp32 || KIND == kXPlanes ? 2 : 1;      // KiB of a unit of one row, each one load of a wavefront
    static constexpr uint32_t kBytes = KIND == kXFp32 ? 4 : 2;                     // of an element, in one array
    // of a column in LDS: 16 bytes more than its data, so that eight neighbouring columns lie in different banks
    static constexpr uint32_t kPitch = 1024 * kLoads + 16;
};

// The rows of x that a wavefront multiplies, on their way through its own piece of LDS (columns * XTraits::kPitch bytes).
// ALIGNED: rows of x start at multiples of 16 bytes, and need not pass through registers.
template <int KIND, bool ALIGNED>
struct XColumns {
    using T = XTraits<KIND>;
    const uint8_t* x;
    size_t pitch, plane;       // bytes
    uint32_t row_bytes;        // k elements of one array
    uint32_t columns;          // 1 to 16
    uint32_t row;              // lane c: the row of x that is column c
    uint8_t* lds;

    // a unit of every column to LDS; what lies past the end of a row is not read
    __device__ __forceinline__ void fetch(uint32_t unit) const {
        const uint32_t lane = threadIdx.x & 63;
        for (uint32_t c = 0; c < columns; ++c) {
            const uint8_t* const r = x + (size_t)__builtin_amdgcn_readlane(row, c) * pitch;
#pragma unroll
            for (int i = 0; i < T::kLoads; ++i) {
                const uint8_t* const p = r + (KIND == kXPlanes && i ? plane : 0);
                const uint32_t at = unit * (kUnitK * T::kBytes) + (KIND == kXFp32 ? i * 1024 : 0) + lane * 16;
                uint8_t* const to = lds + c * T::kPitch + i * 1024;
                if constexpr (ALIGNED) {
                    const auto row_only = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, row_bytes, 0x00020000);
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(row_only, (__attribute__((address_space(3))) void*)to, 16, at, 0, 0, 0);
                } else {
                    uint4 v;
                    __builtin_memcpy(&v, p + min(at, row_bytes - 16), 16);
                    *reinterpret_cast<uint4*>(to + lane * 16) = v;
                }
            }
        }
    }
    // values [8 j, 8 j + 8) of this lane's block of a step as kPieces operands.  A value is the sum of its pieces, exactly: each takes the leading eight
    // bits of what is left.
    __device__ __forceinline__ void operands(uint32_t my_column, int step, int j, bool live, v8bf16 (&out)[T::kPieces]) const {
        const uint32_t q = (threadIdx.x & 63) >> 4;
        const uint8_t* const p = lds + my_column * T::kPitch + ((step * 4 + q) * 4 + j) * (8 * T::kBytes);
        uint4 a = *reinterpret_cast<const uint4*>(p), b = make_uint4(0, 0, 0, 0);
        if constexpr (T::kLoads == 2) b = *reinterpret_cast<const uint4*>(p + (KIND == kXPlanes ? 1024 : 16));
        if (!live) a = b = make_uint4(0, 0, 0, 0);
        if constexpr (KIND == kXBf16) {
            out[0] = __builtin_bit_cast(v8bf16, a);
        } else if constexpr (KIND == kXPlanes) {
            out[0] = __builtin_bit_cast(v8bf16, a);
            out[1] = __builtin_bit_cast(v8bf16, b);
        } else {
            float v[8];
            if constexpr (KIND == kXFp16) {
                typedef _Float16 v8f16 __attribute__((ext_vector_type(8)));
                const v8f16 h = __builtin_bit_cast(v8f16, a);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
            } else {
                const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
            }
#pragma unroll
            for (int p = 0; p < T::kPieces; ++p) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = __builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);      // upper halves
                out[p] = __builtin_bit_cast(v8bf16, make_uint4(w[0], w[1], w[2], w[3]));
                if (p + 1 < T::kPieces) {
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
// byte `i` of a word of E8M0 scales -> the float that scales a conversion: 2^(byte - 127), NaN for 255
__device__ __forceinline__ float e8m0_value(uint32_t word, int i) {
    const uint32_t byte = word >> (8 * i) & 0xFFu;
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

// The lanes of quarter g of a wavefront hold the four scales of step g of their row; afterwards they hold those of block g of each of the four steps: a
// 4 x 4 transposition of bytes across quarters, two lane exchanges and two byte permutations.
__device__ __forceinline__ uint32_t scales_by_block(uint32_t word) {
    const uint32_t g = (threadIdx.x & 63) >> 4;
    const auto far = __builtin_amdgcn_permlane32_swap(word, word, false, false);         // steps g & 1, (g & 1) + 2
    const uint32_t pairs = __builtin_amdgcn_perm(far[1], far[0], g | (g ^ 1) << 8 | (4 + g) << 16 | (4 + (g ^ 1)) << 24);
    const auto near = __builtin_amdgcn_permlane16_swap(pairs, pairs, false, false);      // of the even quarter, of the odd one
    return __builtin_amdgcn_perm(near[1], near[0], (g & 1) ? 0x06030401u : 0x07020500u);
}

// ---- the tile -------------------------------------------------------------------------------------------------------
// RT x 16 weight rows times up to 16 activation rows.  The pointers are a lane's own: weight row l % 16 of each row tile at block l / 16, its scales
// at their start.  blocks: K / 32.
template <int KIND, int RT>
struct RowsTile {
    const uint8_t *a[RT], *scale[RT];
    uint32_t blocks;
    v4f acc[RT];

    struct Regs {
        uint4 a[RT][kUnitSteps];
        uint32_t scale[RT];
    };

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i] = (v4f){0, 0, 0, 0};
    }
    __device__ __forceinline__ void load(Regs& g, uint32_t unit) const {
        const uint32_t q = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            __builtin_memcpy(&g.scale[i], scale[i] + unit * kUnitBlocks + q * 4, 4);
#pragma unroll
            for (int s = 0; s < (int)kUnitSteps; ++s) g.a[i][s] = *reinterpret_cast<const uint4*>(a[i] + ((size_t)unit * kUnitSteps + s) * 64);
        }
    }
    // the unit that K ends in; blocks past the last: codes of zero under a scale of one
    __device__ __forceinline__ void load_end(Regs& g, uint32_t unit) const {
        const uint32_t q = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            g.scale[i] = 0x7F7F7F7Fu;
            for (uint32_t b = 0; b < 4; ++b) {
                const uint32_t at = unit * kUnitBlocks + q * 4 + b;
                if (at < blocks) g.scale[i] = (g.scale[i] & ~(0xFFu << (8 * b))) | (uint32_t)scale[i][at] << (8 * b);
            }
#pragma unroll
            for (int s = 0; s < (int)kUnitSteps; ++s) {
                const uint32_t step = unit * kUnitSteps + s;
                g.a[i][s] = make_uint4(0, 0, 0, 0);
                if (step * 4 + q < blocks) g.a[i][s] = *reinterpret_cast<const uint4*>(a[i] + (size_t)step * 64);
            }
        }
    }
    template <bool WHOLE, bool ALIGNED>
    __device__ __forceinline__ void multiply(const Regs& g, const XColumns<KIND, ALIGNED>& x, uint32_t unit, uint32_t my_column) {
        const uint32_t q = (threadIdx.x & 63) >> 4;
        uint32_t by_block[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) by_block[i] = scales_by_block(g.scale[i]);
#pragma unroll
        for (int s = 0; s < (int)kUnitSteps; ++s) {
            const bool live = WHOLE || (unit * kUnitSteps + s) * 4 + q < blocks;
            float f[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) f[i] = e8m0_value(by_block[i], s);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v8bf16 xs[XTraits<KIND>::kPieces];
                x.operands(my_column, s, j, live, xs);
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const uint4 c = g.a[i][s];
                    const v8bf16 w = e2m1_to_bf16(j == 0 ? c.x : (j == 1 ? c.y : (j == 2 ? c.z : c.w)), f[i]);
#pragma unroll
                    for (int p = 0; p < XTraits<KIND>::kPieces; ++p) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, xs[p], acc[i], 0, 0, 0);
                }
            }
        }
    }
    // Units first, first + by, ... below last.  The weights of a unit are under way while the one before it is multiplied; its activations are requested when
    // that is done, since they go to the same LDS.  (Nothing in the loop is conditional: the wait in front of the reads from LDS
    // then leaves the loads that were issued after the activations' in flight.)
    template <bool ALIGNED>
    __device__ __forceinline__ void run(const XColumns<KIND, ALIGNED>& x, uint32_t first, uint32_t last, uint32_t by) {
        const uint32_t my_column = min(threadIdx.x & 15, x.columns - 1);      // (columns past the last repeat it)
        const uint32_t end = min(last, blocks / kUnitBlocks);                 // of the whole units
        if (first < end) {
            Regs g[2];                                                        // (by turns: a copy would wait for what it copies)
            uint32_t u = first;
            const auto turn = [&](const Regs& now, Regs& next) {
                load(next, u + by);
                __builtin_amdgcn_sched_barrier(0);                            // (they stay in front of the work)
                multiply<true>(now, x, u, my_column);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");            // the reads of this unit are done
                x.fetch(u + by);
                u += by;
            };
            x.fetch(first);
            load(g[0], first);
            bool odd = false;
            while (u + by < end) {
                turn(g[0], g[1]);
                if (u + by >= end) {
                    odd = true;
                    break;
                }
                turn(g[1], g[0]);
            }
            if (odd) multiply<true>(g[1], x, u, my_column);
            else multiply<true>(g[0], x, u, my_column);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            first = u + by;
        }
        if (first < last) {
            Regs g;
            x.fetch(first);
            load_end(g, first);
            multiply<false>(g, x, first, my_column);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
};

}  // namespace cmx
