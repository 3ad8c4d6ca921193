// A few rows of 16- or 32-bit activations times MXFP4 weights: the work of one wavefront.
//
// The weights are the matrix instruction's rows: v_mfma_f32_16x16x32_bf16 takes 16 weight rows and up to 16 activation rows as its
// columns.  E2M1 times a power of two is exact in bf16 and an activation is one bf16 value or a sum of two or three (fp16, fp32), so
// every product is exact and sums are fp32: nothing is rounded before the result.  Which K a lane's eight values stand for is free as long as
// both operands agree, so that a lane's share of a step is 16 bytes of its weight row = 32 codes = one block with one scale, feeding four
// instructions.  Lane l: row (or column) l % 16, block l / 16 of the step's four.
//
// What bounds this on the way to the memory's rate is the address path of a CU, where a load of a wavefront costs about as many cycles as it touches
// pieces of memory, and the bytes in flight.  Weights loaded as the instruction wants them (16 rows, 16 bytes per lane, neighbouring lanes in
// different rows) touch 64 pieces, scale bytes and activations as many again.  So everything is loaded as it lies - four rows x 256 bytes of weights,
// 16 bytes of a row's scales, whole kilobytes of activations - into registers, of which a CU has three times as much as LDS, and changes lanes through a
// piece of LDS that is the wavefront's own: nothing waits for another wavefront.
// Measured (both matmuls of the FFN of 32 tokens, 163 of 256 experts with 3.8 GB of weights, K = 7168, N = 4096; us): loads as the instruction wants them, a
// scale byte per lane and step, 1541; scales by the word and activations straight to LDS 930; everything as it lies 745.  Of that the first matmul reads
// at 5.7 TB/s and the second at 4.2; a plain sum over as many bytes reaches 6.2.
#pragma once

#include "mx_common.h"

namespace cmx {

typedef __bf16 v8bf16 __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr uint32_t kUnitSteps = 4, kUnitBlocks = 16, kUnitK = 512;        // a step: four blocks of 32 along K, one for each 16 lanes

// ---- activations ----------------------------------------------------------------------------------------------------
// kXPlanes: two bf16 arrays, `plane` bytes apart, whose sum is the value
enum XKind { kXBf16 = CMX_OUT_BF16, kXFp16 = CMX_OUT_FP16, kXFp32 = CMX_OUT_FP32, kXPlanes = 3 };

template <int KIND>
struct XTraits {
    static constexpr int kPieces = KIND == kXBf16 ? 1 : (KIND == kXFp32 ? 3 : 2);
    static constexpr uint32_t kBytes = KIND == kXFp32 ? 4 : 2;                     // of an element, in one array
    static constexpr int kReads = KIND == kXFp32 || KIND == kXPlanes ? 2 : 1;      // 16-byte pieces that hold eight values
};
// Whether fp16 and fp32 are taken to pieces on their way into LDS, once for each value, or behind it, by each lane that takes it: a tile's 16 columns are
// COLUMNS rows of x again and again.  Pieces take more of LDS than the value, which costs wavefronts where columns are many.  (Matrix-vector product,
// 4096 x 7168, us, behind LDS and before: fp16, 1 row 10.8 and 7.0, 8 rows 12.2 and 10.1; fp32, 1 row 13.4 and 8.1, 8 rows 16.4 and 14.5.)
template <int KIND, int COLUMNS>
constexpr bool kPiecesInLds = KIND == kXPlanes || KIND == kXFp32 || (KIND == kXFp16 && COLUMNS <= 8);
// 16-byte parts of LDS that hold eight values: of each piece, or of the value
template <int KIND, int COLUMNS>
constexpr int kParts = kPiecesInLds<KIND, COLUMNS> ? XTraits<KIND>::kPieces : XTraits<KIND>::kReads;
// bytes of a column in LDS: a unit of one row of x
template <int KIND, int COLUMNS>
constexpr uint32_t kColumnPitch = kParts<KIND, COLUMNS> * 1024 + 16;

__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p; }
// ---- weights --------------------------------------------------------------------------------------------------------
// E8M0 byte -> the float that scales a conversion: 2^(byte - 127), NaN for 255
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    const uint32_t bits = byte == 0 ? 0x00400000u : byte << 23;
    return __uint_as_float(byte == 255 ? 0x7FC00000u : bits);
}

// eight E2M1 codes times a scale
__device__ __forceinline__ v8bf16 e2m1_to_bf16(uint32_t codes, float scale) {
    v4u w;
    w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    w.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    w.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    return __builtin_bit_cast(v8bf16, w);
}

// ---- the wavefront --------------------------------------------------------------------------------------------------
constexpr uint32_t kRowPitch = 256 + 16;        // of a weight row in LDS

// Bytes of LDS of a wavefront: a unit of RT x 16 weight rows, 16 bytes of scales for each, COLUMNS columns of activations
template <int KIND, int RT, int COLUMNS>
constexpr uint32_t kStageBytes = RT * (16 * kRowPitch + 256) + COLUMNS * kColumnPitch<KIND, COLUMNS>;

// RT x 16 weight rows times up to COLUMNS (1 to 16) activation rows.
//
// The lanes of a read from LDS want the same 16-byte piece of 16 rows (columns): 16 bytes between these put eight neighbours into different banks.
// STREAM: weights that are read once pass by the caches, which keep the activations.
template <int KIND, int RT, int COLUMNS, bool STREAM>
struct RowsStream {
    using T = XTraits<KIND>;
    static constexpr bool kInPieces = kPiecesInLds<KIND, COLUMNS>;
    static constexpr int kPartsOf = kParts<KIND, COLUMNS>;
    static constexpr uint32_t kPitch = kColumnPitch<KIND, COLUMNS>;
    // a lane's own: where its 16 bytes of each group of four weight rows and its four of the scales come from, at K = 0
    const uint8_t *a[RT][4], *scale[RT];
    uint32_t blocks;           // K / 32
    const uint8_t* x;
    size_t x_pitch, plane;     // bytes
    uint32_t row;              // lane c: the row of x that is column c, up to COLUMNS
    uint32_t stage;            // LDS address
    v4f acc[RT][T::kPieces];   // one for each piece: products that do not wait for each other

    // a unit on its way
    struct Unit {
        v4u a[RT][4], x[COLUMNS][T::kReads];
        uint32_t scale[RT];
    };

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int n = 0; n < T::kPieces; ++n) acc[i][n] = (v4f){0, 0, 0, 0};
    }
    __device__ __forceinline__ v4f sum(int i) const {
        v4f v = acc[i][0];
#pragma unroll
        for (int n = 1; n < T::kPieces; ++n) v += acc[i][n];
        return v;
    }
    // Row tile i: 16 rows from `first` on, of which those past `last` are taken for `last`; the arrays' pitches in bytes.
    __device__ __forceinline__ void set_rows(int i, const uint8_t* codes, size_t pitch, const uint8_t* scales, size_t scale_pitch, uint32_t first, uint32_t last) {
        const uint32_t lane = threadIdx.x & 63;
#pragma unroll
        for (int g = 0; g < 4; ++g) a[i][g] = codes + min(first + g * 4 + lane / 16, last) * pitch + lane % 16 * 16;
        scale[i] = scales + min(first + lane / 4, last) * scale_pitch + lane % 4 * 4;
    }
    __device__ __forceinline__ bool whole(uint32_t unit) const { return (unit + 1) * kUnitBlocks <= blocks; }      // the same for every lane

    // what lies past the end of a row is not read
    __device__ __forceinline__ void load(Unit& u, uint32_t unit) const {
        const uint32_t lane = threadIdx.x & 63, row_bytes = blocks * 32 * T::kBytes;
        const bool all = whole(unit);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (all) {
                __builtin_memcpy(&u.scale[i], scale[i] + (size_t)unit * kUnitBlocks, 4);
            } else {
                u.scale[i] = 0;
#pragma unroll
                for (uint32_t b = 0; b < 4; ++b)
                    if (unit * kUnitBlocks + lane % 4 * 4 + b < blocks) u.scale[i] |= (uint32_t)scale[i][unit * kUnitBlocks + b] << (8 * b);
            }
            const uint32_t block = unit * kUnitBlocks + lane % 16, back = all || block < blocks ? 0 : (block - (blocks - 1)) * 16;      // (its last block instead)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const v4u* const p = reinterpret_cast<const v4u*>(a[i][g] + (size_t)unit * 256 - back);
                u.a[i][g] = STREAM ? __builtin_nontemporal_load(p) : *p;
            }
        }
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) {
            const uint8_t* const r = x + (size_t)__builtin_amdgcn_readlane(row, c) * x_pitch;
#pragma unroll
            for (int l = 0; l < T::kReads; ++l) {
                const uint32_t off = min(unit * (kUnitK * T::kBytes) + (KIND == kXFp32 ? l * 1024 : 0) + lane * 16, row_bytes - 16);
                __builtin_memcpy(&u.x[c][l], r + off + (KIND == kXPlanes && l ? plane : 0), 16);
            }
        }
    }
    __device__ __forceinline__ void store(const Unit& u) const {
        typedef __attribute__((address_space(3))) v4u* lds4;
        const uint32_t lane = threadIdx.x & 63, xs = stage + RT * (16 * kRowPitch + 256);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            *(__attribute__((address_space(3))) uint32_t*)(uintptr_t)(stage + RT * (16 * kRowPitch) + i * 256 + lane * 4) = u.scale[i];
#pragma unroll
            for (int g = 0; g < 4; ++g) *(lds4)(uintptr_t)(stage + (i * 16 + g * 4 + lane / 16) * kRowPitch + lane % 16 * 16) = u.a[i][g];
        }
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) {
            const uint32_t to = xs + c * kPitch + lane * 16;
            if constexpr (!kInPieces || KIND == kXPlanes) {
#pragma unroll
                for (int l = 0; l < T::kReads; ++l) *(lds4)(uintptr_t)(to + l * 1024) = u.x[c][l];
            } else if constexpr (KIND == kXFp16) {
                v8bf16 piece[T::kPieces];
                operands(&u.x[c][0], piece);
#pragma unroll
                for (int n = 0; n < T::kPieces; ++n) *(lds4)(uintptr_t)(to + n * 1024) = __builtin_bit_cast(v4u, piece[n]);
            } else {
                typedef __attribute__((address_space(3))) v2u* lds2;      // (four of the eight values from each half of the unit)
                v8bf16 piece[T::kPieces];
                operands(&u.x[c][0], piece);
#pragma unroll
                for (int n = 0; n < T::kPieces; ++n) {
                    const v4u w = __builtin_bit_cast(v4u, piece[n]);
                    *(lds2)(uintptr_t)(to - lane * 8 + n * 1024) = (v2u){w.x, w.y};
                    *(lds2)(uintptr_t)(to - lane * 8 + n * 1024 + 512) = (v2u){w.z, w.w};
                }
            }
        }
    }

    // what a lane takes from LDS for one step
    struct Step {
        v4u codes[RT], x[4][kPartsOf];
        uint32_t scale[RT];
    };
    __device__ __forceinline__ void read(Step& g, uint32_t xs, int s) const {
        typedef const __attribute__((address_space(3))) v4u* lds4;
        typedef const __attribute__((address_space(3))) uint8_t* lds1;
        constexpr uint32_t kBytes = kInPieces ? 2 : T::kBytes;
        const uint32_t r = threadIdx.x & 15, q = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            g.codes[i] = *(lds4)(uintptr_t)(stage + (i * 16 + r) * kRowPitch + q * 16 + s * 64);
            g.scale[i] = *(lds1)(uintptr_t)(stage + RT * (16 * kRowPitch) + i * 256 + r * 16 + q + s * 4);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int l = 0; l < kPartsOf; ++l)
                g.x[j][l] = *(lds4)(uintptr_t)(xs + q * (32 * kBytes) + s * (128 * kBytes) + j * (8 * kBytes) + l * 1024);
    }
    // eight activations as kPieces operands.  A value is the sum of its pieces, exactly: each takes the leading eight bits of what is left.
    __device__ __forceinline__ static void operands(const v4u* x, v8bf16 (&out)[T::kPieces]) {
        if constexpr (KIND == kXBf16) {
            out[0] = __builtin_bit_cast(v8bf16, x[0]);
        } else if constexpr (KIND != kXPlanes) {
            float v[8];
            if constexpr (KIND == kXFp16) {
                typedef _Float16 v8f16 __attribute__((ext_vector_type(8)));
                const v8f16 h = __builtin_bit_cast(v8f16, x[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
            } else {
                const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
            }
#pragma unroll
            for (int n = 0; n < T::kPieces; ++n) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = __builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);      // upper halves
                out[n] = __builtin_bit_cast(v8bf16, (v4u){w[0], w[1], w[2], w[3]});
                if (n + 1 < T::kPieces) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float lead = __uint_as_float(__float_as_uint(v[i]) & 0xFFFF0000u);
                        v[i] = lead == v[i] ? 0.0f : v[i] - lead;          // (Inf leaves nothing, a NaN a NaN)
                    }
                }
            }
        }
    }
    // the unit in LDS, onto acc
    template <bool WHOLE>
    __device__ __forceinline__ void multiply(uint32_t unit) {
        const uint32_t q = (threadIdx.x & 63) >> 4, xs = stage + RT * (16 * kRowPitch + 256) + (threadIdx.x & 15) % COLUMNS * kPitch;      // (columns again and again)
#pragma unroll
        for (int s = 0; s < (int)kUnitSteps; ++s) {
            Step g;
            read(g, xs, s);
            if (!WHOLE && (unit * kUnitSteps + s) * 4 + q >= blocks) {      // past the end of K: zeros on both sides
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    g.codes[i] = (v4u){0, 0, 0, 0};
                    g.scale[i] = 127;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int l = 0; l < kPartsOf; ++l) g.x[j][l] = (v4u){0, 0, 0, 0};
            }
            float f[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) f[i] = e8m0_value(g.scale[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v8bf16 v[T::kPieces];
                if constexpr (kInPieces) {
#pragma unroll
                    for (int n = 0; n < T::kPieces; ++n) v[n] = __builtin_bit_cast(v8bf16, g.x[j][n]);
                } else {
                    operands(g.x[j], v);
                }
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const v4u c = g.codes[i];
                    const v8bf16 w = e2m1_to_bf16(j == 0 ? c.x : (j == 1 ? c.y : (j == 2 ? c.z : c.w)), f[i]);
#pragma unroll
                    for (int n = 0; n < T::kPieces; ++n) acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, v[n], acc[i][n], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);                              // (or the reads of all steps are held at once)
        }
    }
    // One turn: the unit that was loaded goes to LDS, the next is requested (unless there is none), the one in LDS is multiplied.
    template <class Next>
    __device__ __forceinline__ void turn(Unit& u, uint32_t unit, const Next& load_next) {
        store(u);
        load_next(u);
        __builtin_amdgcn_sched_barrier(0);                                  // (the loads stay in front of the work)
        __builtin_amdgcn_wave_barrier();
        if (whole(unit)) multiply<true>(unit);
        else multiply<false>(unit);
        __builtin_amdgcn_wave_barrier();
    }
    // units first, first + by, ... below last
    __device__ __forceinline__ void run(uint32_t first, uint32_t last, uint32_t by) {
        if (first >= last) return;
        Unit u;
        load(u, first);
        for (uint32_t n = first; n < last; n += by)
            turn(u, n, [&](Unit& v) {
                if (n + by < last) load(v, n + by);
            });
    }
};

}  // namespace cmx
