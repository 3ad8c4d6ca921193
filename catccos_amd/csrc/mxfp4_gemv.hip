// out[m, n] = x[m, k] . deq(b)[n, k]^T for few rows of x: a matrix-vector product and a little more, bound by reading the weights once.
//
// A workgroup owns RT x 16 weight rows over the whole of K, which its wavefronts share out unit by unit; their sums meet in LDS.
// Measured, bf16 x, weights from memory: one row of x, 16384 x 8192 in 18.6 us (3.8 TB/s), 4096 x 7168 in 6.1 us (2.6 TB/s: start, one wait for memory and the
// join are 4 of them).
#include "mx_launch.h"
#include "mxfp4_rows.h"

namespace cmx {
namespace {

struct GemvArgs {
    const uint8_t *x, *b, *b_scale;
    uint8_t* out;
    size_t ld_x, ld_b, ld_scale, ld_out;      // bytes
    uint32_t m, n, blocks;
    int out_type;
};

// four consecutive results, or as many as `left`, to p
__device__ __forceinline__ void store4(uint8_t* p, const v4f v, int type, uint32_t left) {
    uint32_t w[4];
    if (type == CMX_OUT_FP32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
        if (left >= 4) __builtin_memcpy(p, w, 16);
        else
            for (uint32_t i = 0; i < left; ++i) reinterpret_cast<float*>(p)[i] = v[i];
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
    if (left >= 4) {
        __builtin_memcpy(p, w, 8);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
        if (i < left) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
}

// wavefronts of a workgroup: more than 8 where registers and LDS allow (one row of x, 336 x 13024: 6.0 us, with 8 6.8; 4096 x 7168 the same 6.1)
template <int COLUMNS>
constexpr uint32_t kGemvWaves = COLUMNS <= 4 ? 12 : 8;

template <int KIND, int RT, int COLUMNS>
__global__ __launch_bounds__(64 * kGemvWaves<COLUMNS>) void mxfp4_gemv_kernel(const GemvArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // a stage for each wavefront, then sums: [wavefront][row tile][lane]
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t row0 = blockIdx.x * (16 * RT), col0 = blockIdx.y * COLUMNS;
    RowsStream<KIND, RT, COLUMNS, false> t;
    t.blocks = a.blocks;
#pragma unroll
    for (int i = 0; i < RT; ++i) t.set_rows(i, a.b, a.ld_b, a.b_scale, a.ld_scale, row0 + i * 16, a.n - 1);      // (rows past the last are not stored)
    t.x = a.x;
    t.x_pitch = a.ld_x;
    t.plane = 0;
    t.row = min(col0 + lane, a.m - 1);
    t.stage = lds_address(lds) + wave * kStageBytes<KIND, RT, COLUMNS>;
    t.clear();
    t.run(wave, (a.blocks + kUnitBlocks - 1) / kUnitBlocks, waves);
    __syncthreads();
    v4f* const sums = reinterpret_cast<v4f*>(lds);
#pragma unroll
    for (int i = 0; i < RT; ++i) sums[(wave * RT + i) * 64 + lane] = t.sum(i);
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < RT * 64; at += blockDim.x) {
        v4f v = sums[at];
        for (uint32_t w = 1; w < waves; ++w) v += sums[w * (RT * 64) + at];
        const uint32_t l = at & 63, i = at >> 6;
        const uint32_t row = row0 + i * 16 + (l >> 4) * 4, col = l & 15;     // of weights: output columns; of x: output rows
        if (row < a.n && col < COLUMNS && col0 + col < a.m)
            store4(a.out + (col0 + col) * a.ld_out + (size_t)row * (a.out_type == CMX_OUT_FP32 ? 4 : 2), v, a.out_type, a.n - row);
    }
}

template <int KIND, int RT, int COLUMNS>
int launch(const GemvArgs& a, hipStream_t s) {
    constexpr uint32_t kEach = kStageBytes<KIND, RT, COLUMNS>, kFit = 160 * 1024 / kEach, kMaxWaves = kFit < kGemvWaves<COLUMNS> ? kFit : kGemvWaves<COLUMNS>;
    // as many wavefronts as share the units of K evenly
    const uint32_t units = ceil_div(a.blocks, kUnitBlocks), waves = ceil_div(units, ceil_div(units, kMaxWaves));
    if (int rc = allow_dynamic_lds<mxfp4_gemv_kernel<KIND, RT, COLUMNS>, kMaxWaves * kEach>(); rc != CMX_OK) return rc;
    hipLaunchKernelGGL((mxfp4_gemv_kernel<KIND, RT, COLUMNS>), dim3(ceil_div(a.n, 16 * RT), ceil_div(a.m, COLUMNS)), dim3(64 * waves), waves * kEach, s, a);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

// Two tiles of rows share what a workgroup reads of x, one tile makes twice the workgroups.  Up to 4 rows of x the workgroups matter more (us, bf16 x, weights
// from memory, one tile / two tiles, N x K: 1 row of x, 4096 x 7168 6.1 / 7.5, 16384 x 8192 18.6 / 20.8; 4 rows, 32768 x 2048 10.4 / 12.0); from 5 rows on
// two tiles win where they still leave three workgroups to four CUs (8 rows, 16384 x 8192 28.4 / 23.2; 16 rows, 7168 x 2048 7.9 / 5.3, 16384 x 8192
// 34.6 / 26.0; 64 rows, 4096 x 7168 25.8 / 18.0) and lose where they do not (8 rows, 4096 x 7168 7.6 / 9.5; 16 rows 9.6 / 10.9, 2048 x 16384 14.6 / 18.7).
// Four tiles spill registers or take too much LDS (16 rows, 16384 x 8192: 44).
template <int KIND, int COLUMNS>
int launch_tiles(const GemvArgs& a, hipStream_t s) {
    int cus;
    if (int rc = cu_count(&cus); rc != CMX_OK) return rc;
    if (4 * (uint64_t)ceil_div(a.n, 32) * ceil_div(a.m, COLUMNS) >= 3 * (uint64_t)cus) return launch<KIND, 2, COLUMNS>(a, s);
    return launch<KIND, 1, COLUMNS>(a, s);
}

template <int KIND>
int launch(const GemvArgs& a, hipStream_t s) {
    constexpr uint32_t kMost = KIND == kXFp32 ? 8 : 16;
    int cus;
    if (int rc = cu_count(&cus); rc != CMX_OK) return rc;
    uint32_t columns = 1;
    while (columns < kMost && columns < a.m) columns *= 2;
    // A long K under few weight rows: workgroups that share a weight row's tile have fewer columns each, which costs them less time than the CUs stood idle
    // (K > 4096; 16 columns / as many as leave a workgroup to a CU, 16 rows of x: 127 x 15584 bf16 11.7 / 7.1 us, fp16 21.7 / 9.1, fp32 26.5 / 10.8,
    // 728 x 11424 bf16 10.8 / 7.4; up to K = 4096 a wavefront has one unit and nothing is gained: 1756 x 896 3.9 / 4.3).
    while (columns > 1 && a.blocks > 8 * kUnitBlocks && (uint64_t)ceil_div(a.n, 16) * ceil_div(a.m, columns / 2) <= (uint32_t)cus) columns /= 2;
    if (columns <= 1) return launch<KIND, 1, 1>(a, s);
    if (columns <= 2) return launch<KIND, 1, 2>(a, s);
    if (columns <= 4) return launch<KIND, 1, 4>(a, s);
    if (columns <= 8 || kMost == 8) return launch_tiles<KIND, 8>(a, s);
    // fp16: 8 columns come out of LDS in pieces, 16 have to be split behind it (16 rows of x, 4096 x 7168: one tile of rows and 16 columns 14.0 us, two and
    // 8 11.9; 5120 x 8192 27.7 and 21.4; with two tiles under both, 24 rows of 4096 x 7168, 16 columns 16.7 and 8 20.6).
    if constexpr (KIND == kXFp16) {
        const auto two_tiles = [&](uint32_t by) { return 4 * (uint64_t)ceil_div(a.n, 32) * ceil_div(a.m, by) >= 3 * (uint64_t)cus; };
        if (!two_tiles(16) && two_tiles(8)) return launch<KIND, 2, 8>(a, s);
    }
    return launch_tiles<KIND, kMost>(a, s);
}

}  // namespace
}  // namespace cmx

int cmx::preload_gemv_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::mxfp4_gemv_kernel<kXBf16, 1, 1>)));
    return CMX_OK;
}

extern "C" int cmx_mxfp4_gemv(const void* x, uint32_t ld_x, int x_type, const uint8_t* b, uint32_t ld_b, const uint8_t* b_scale, uint32_t ld_bs,
                              void* out, uint32_t ld_out, int out_type, uint32_t m, uint32_t n, uint32_t k, cmx_stream_t stream) {
    using namespace cmx;
    const auto known = [](int t) { return t == CMX_OUT_BF16 || t == CMX_OUT_FP16 || t == CMX_OUT_FP32; };
    CMX_REQUIRE(known(x_type) && known(out_type), "unknown type");
    if (m == 0 || n == 0) return CMX_OK;
    CMX_REQUIRE(x && b && b_scale && out, "null pointer");
    CMX_REQUIRE(k > 0 && k % 32 == 0 && k <= (1u << 29), "k must be a positive multiple of 32, at most 2^29");
    CMX_REQUIRE(n <= (1u << 26), "too many rows of b");
    CMX_REQUIRE(ld_x >= k && ld_b >= k / 2 && ld_bs >= k / 32 && ld_out >= n, "row pitch smaller than row");
    CMX_REQUIRE(aligned16(b) && ld_b % 16 == 0, "weight rows must be 16-byte aligned");
    const uint32_t xb = x_type == CMX_OUT_FP32 ? 4 : 2, ob = out_type == CMX_OUT_FP32 ? 4 : 2;
    CMX_REQUIRE(reinterpret_cast<uintptr_t>(x) % xb == 0 && reinterpret_cast<uintptr_t>(out) % ob == 0, "pointers must be aligned to their elements");
    CMX_REQUIRE(ceil_div(m, 8) <= 65535u, "too many rows of x");
    const GemvArgs a = {static_cast<const uint8_t*>(x), b, b_scale, static_cast<uint8_t*>(out), (size_t)ld_x * xb, ld_b, ld_bs, (size_t)ld_out * ob, m, n, k / 32,
                        out_type};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (x_type == CMX_OUT_BF16) return launch<kXBf16>(a, s);
    return x_type == CMX_OUT_FP16 ? launch<kXFp16>(a, s) : launch<kXFp32>(a, s);
}
