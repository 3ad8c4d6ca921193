// Token rows to the experts' order, and the gradients of that and of the weighted way back:
//
//   permute          out[dst(t, r)] = x[t]
//   permute_grad     dx[t] = sum_r dy[dst(t, r)]
//   unpermute_grad   dy[dst(t, r)] = probs[t, r] * dout[t],   dprobs[t, r] = sum_h dout[t, h] * y[dst(t, r), h]
//
// with dst(t, r) = src2sorted[t * top_k + r]; a destination outside [0, rows) is a dropped route.  Sums are fp32, of the routes in their order and of h in an order that the
// sizes alone fix.  All are bound by memory: a token's row is read once and kept in registers for its routes.
#include <algorithm>

#include "mx_launch.h"

namespace cmx {
namespace {

constexpr uint32_t kThreads = 256, kMostRoutes = 64, kMapRows = 4096;

// Rows that no route is sent to, cleared by the first workgroups of a launch: each looks through all routes for the `per` rows that it has.
struct ClearJob {
    uint32_t blocks, per, rows, routes;
};
ClearJob clear_job(uint32_t rows, uint32_t routes) {
    const uint32_t per = std::min(kMapRows, round_up(ceil_div(rows, 256u), 32u));
    return {ceil_div(rows, per), per, rows, routes};
}

template <class V>
__device__ __forceinline__ void clear_unmapped_rows(const ClearJob& z, const int32_t* __restrict__ src2sorted, uint8_t* __restrict__ out, size_t ld_out,
                                                    uint32_t vecs) {
    __shared__ uint32_t s_map[kMapRows / 32];
    const uint32_t r0 = blockIdx.x * z.per, n = min(z.per, z.rows - r0), words = (n + 31) / 32;
    for (uint32_t i = threadIdx.x; i < words; i += kThreads) s_map[i] = 0;
    __syncthreads();
    constexpr uint32_t kBatch = 8;
    for (uint64_t i0 = 0; i0 < z.routes; i0 += kBatch * kThreads) {
        int32_t d[kBatch];
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint64_t i = i0 + j * kThreads + threadIdx.x;
            d[j] = i < z.routes ? src2sorted[i] : -1;
        }
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t r = (uint32_t)d[j] - r0;
            if (d[j] >= 0 && (uint32_t)d[j] >= r0 && r < n) atomicOr(&s_map[r / 32], 1u << (r % 32));
        }
    }
    __syncthreads();
    for (uint32_t w = threadIdx.x / 64; w < words; w += kThreads / 64) {
        uint32_t miss = ~s_map[w];
        if (w == words - 1 && n % 32 != 0) miss &= (1u << (n % 32)) - 1u;
        while (miss != 0) {
            V* const row = reinterpret_cast<V*>(out + (size_t)(r0 + w * 32 + (uint32_t)__builtin_ctz(miss)) * ld_out);
            for (uint32_t i = threadIdx.x & 63u; i < vecs; i += 64) row[i] = V{};
            miss &= miss - 1;
        }
    }
}

struct PermuteArgs {
    const uint8_t *x, *dout;              // what is read by rows of the one order and of the other
    const int32_t* src2sorted;
    const float* probs;
    uint8_t* out;
    float* dprobs;
    size_t ld_x, ld_dout, ld_out;         // bytes
    uint32_t tokens, top_k, rows, vecs;
    ClearJob clear;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A lane per (token, V), numbered token-major (a launch has fewer than 2^32).  The copies go past the caches: nothing here reads them again.  8192 tokens of 7168
// bf16, 8 routes: 1.06 GB in 212 us, 5.0 TB/s, the rate of a copy.
template <class V>
__global__ __launch_bounds__(kThreads) void moe_permute_kernel(const PermuteArgs p) {
    if (blockIdx.x < p.clear.blocks) {
        clear_unmapped_rows<V>(p.clear, p.src2sorted, p.out, p.ld_out, p.vecs);
        return;
    }
    const uint32_t item = (blockIdx.x - p.clear.blocks) * kThreads + threadIdx.x, t = item / p.vecs, v = item - t * p.vecs;
    if (t >= p.tokens) return;
    const V value = reinterpret_cast<const V*>(p.x + t * p.ld_x)[v];
    const int32_t* const idx = p.src2sorted + (size_t)t * p.top_k;
    for (uint32_t r0 = 0; r0 < p.top_k; r0 += 8) {
        int32_t d[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) d[j] = r0 + j < p.top_k ? idx[r0 + j] : -1;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (d[j] >= 0 && (uint32_t)d[j] < p.rows) __builtin_nontemporal_store(value, reinterpret_cast<V*>(p.out + d[j] * p.ld_out) + v);
    }
}

// N elements of a type in a register piece V
template <int TYPE, class V>
struct Elements {
    static constexpr uint32_t kSize = TYPE == CMX_OUT_FP32 ? 4 : 2, N = sizeof(V) / kSize;
    __device__ static __forceinline__ void unpack(const V& v, float (&f)[N]) {
        if constexpr (TYPE == CMX_OUT_FP32) __builtin_memcpy(f, &v, sizeof v);
        else {
            uint16_t h[N];
            __builtin_memcpy(h, &v, sizeof v);
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) f[i] = TYPE == CMX_OUT_BF16 ? bf16_to_f32(h[i]) : (float)__builtin_bit_cast(_Float16, h[i]);
        }
    }
    __device__ static __forceinline__ V pack(const float (&f)[N]) {
        V v;
        if constexpr (TYPE == CMX_OUT_FP32) __builtin_memcpy(&v, f, sizeof v);
        else {
            uint16_t h[N];
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) h[i] = TYPE == CMX_OUT_BF16 ? (uint16_t)__builtin_bit_cast(uint16_t, (__bf16)f[i]) : __builtin_bit_cast(uint16_t, (_Float16)f[i]);
            __builtin_memcpy(&v, h, sizeof v);
        }
        return v;
    }
};

// The same shape; eight rows are asked for before the first is added
template <int TYPE, class V>
__global__ __launch_bounds__(kThreads) void moe_permute_grad_kernel(const PermuteArgs p) {
    using E = Elements<TYPE, V>;
    const uint32_t item = blockIdx.x * kThreads + threadIdx.x, t = item / p.vecs, v = item - t * p.vecs;
    if (t >= p.tokens) return;
    const int32_t* const idx = p.src2sorted + (size_t)t * p.top_k;
    float sum[E::N];
#pragma unroll
    for (uint32_t i = 0; i < E::N; ++i) sum[i] = 0.0f;
    for (uint32_t r0 = 0; r0 < p.top_k; r0 += 8) {
        int32_t d[8];
        V raw[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) d[j] = r0 + j < p.top_k ? idx[r0 + j] : -1;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            raw[j] = d[j] >= 0 && (uint32_t)d[j] < p.rows ? __builtin_nontemporal_load(reinterpret_cast<const V*>(p.x + d[j] * p.ld_x) + v) : V{};
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            float f[E::N];
            E::unpack(raw[j], f);
#pragma unroll
            for (uint32_t i = 0; i < E::N; ++i) sum[i] += f[i];
        }
    }
    reinterpret_cast<V*>(p.out + t * p.ld_out)[v] = E::pack(sum);
}

// A workgroup per (token, ROUTES of its routes): a piece of dout is read once and meets the same piece of every y, whose dot products stay in registers until the row
// ends.  8192 tokens of 7168 bf16, 8 routes: 2.0 GB in 404 us, 4.95 TB/s.  One route to a workgroup where tokens alone would leave CUs idle.
template <int TYPE, class V, uint32_t ROUTES>
__global__ __launch_bounds__(kThreads) void moe_unpermute_grad_kernel(const PermuteArgs p) {
    using E = Elements<TYPE, V>;
    if (blockIdx.x < p.clear.blocks) {
        clear_unmapped_rows<V>(p.clear, p.src2sorted, p.out, p.ld_out, p.vecs);
        return;
    }
    __shared__ float s_dot[kThreads / 64][ROUTES];
    const uint32_t parts = (p.top_k + ROUTES - 1) / ROUTES, block = blockIdx.x - p.clear.blocks, t = block / parts, r0 = block % parts * ROUTES;
    const size_t route = (size_t)t * p.top_k + r0;
    int32_t d[ROUTES];
    float w[ROUTES], dot[ROUTES];
    bool in[ROUTES];
#pragma unroll
    for (uint32_t j = 0; j < ROUTES; ++j) {
        const bool there = r0 + j < p.top_k;
        d[j] = there ? p.src2sorted[route + j] : -1;
        w[j] = there ? p.probs[route + j] : 0.0f;
        in[j] = d[j] >= 0 && (uint32_t)d[j] < p.rows;
        dot[j] = 0.0f;
    }
    for (uint32_t v = threadIdx.x; v < p.vecs; v += kThreads) {
        float g[E::N];
        E::unpack(reinterpret_cast<const V*>(p.dout + t * p.ld_dout)[v], g);
        V raw[ROUTES];
#pragma unroll
        for (uint32_t j = 0; j < ROUTES; ++j)
            if (in[j]) raw[j] = __builtin_nontemporal_load(reinterpret_cast<const V*>(p.x + d[j] * p.ld_x) + v);
#pragma unroll
        for (uint32_t j = 0; j < ROUTES; ++j) {
            if (!in[j]) continue;
            float y[E::N], o[E::N];
            E::unpack(raw[j], y);
#pragma unroll
            for (uint32_t i = 0; i < E::N; ++i) {
                dot[j] = __builtin_fmaf(g[i], y[i], dot[j]);
                o[i] = w[j] * g[i];
            }
            __builtin_nontemporal_store(E::pack(o), reinterpret_cast<V*>(p.out + d[j] * p.ld_out) + v);
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < ROUTES; ++j) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) dot[j] += __shfl_xor(dot[j], o);
        if ((threadIdx.x & 63u) == 0) s_dot[threadIdx.x >> 6][j] = dot[j];
    }
    __syncthreads();
    if (threadIdx.x < ROUTES && r0 + threadIdx.x < p.top_k) {
        float s = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kThreads / 64; ++i) s += s_dot[i][threadIdx.x];
        p.dprobs[route + threadIdx.x] = s;
    }
}

// bytes of the widest pieces that the rows consist of
uint32_t piece_bytes(uint64_t row_bytes, std::initializer_list<uint64_t> addresses_and_pitches) {
    uint64_t all = row_bytes | 16;
    for (uint64_t v : addresses_and_pitches) all |= v;
    return (uint32_t)(all & (~all + 1));
}

template <int TYPE, class V>
int launch_unpermute_grad(PermuteArgs p, hipStream_t s) {
    p.vecs /= Elements<TYPE, V>::N;
    // a workgroup to a route where tokens alone leave CUs idle
    const bool few = (uint64_t)p.tokens * p.top_k <= 2048;
    const uint64_t blocks = p.clear.blocks + (uint64_t)p.tokens * (few ? p.top_k : ceil_div(p.top_k, 8));
    CMX_REQUIRE(fits_grid(blocks, kThreads), "too many tokens");
    if (few) hipLaunchKernelGGL((moe_unpermute_grad_kernel<TYPE, V, 1>), dim3((uint32_t)blocks), dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((moe_unpermute_grad_kernel<TYPE, V, 8>), dim3((uint32_t)blocks), dim3(kThreads), 0, s, p);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

template <int TYPE, class V>
int launch_permute_grad(PermuteArgs p, hipStream_t s) {
    p.vecs /= Elements<TYPE, V>::N;
    const uint64_t blocks = ((uint64_t)p.tokens * p.vecs + kThreads - 1) / kThreads;
    CMX_REQUIRE(fits_grid(blocks, kThreads), "too many elements");
    hipLaunchKernelGGL((moe_permute_grad_kernel<TYPE, V>), dim3((uint32_t)blocks), dim3(kThreads), 0, s, p);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

// f(type constant, piece) for a type and rows of pieces of `bytes`: whole 16-byte pieces, or single elements
template <class F>
int by_type(int type, uint32_t bytes, F&& f) {
    const bool wide = bytes == 16;
    if (type == CMX_OUT_FP32) return wide ? f(std::integral_constant<int, CMX_OUT_FP32>{}, u32x4{}) : f(std::integral_constant<int, CMX_OUT_FP32>{}, uint32_t{});
    if (type == CMX_OUT_FP16) return wide ? f(std::integral_constant<int, CMX_OUT_FP16>{}, u32x4{}) : f(std::integral_constant<int, CMX_OUT_FP16>{}, uint16_t{});
    return wide ? f(std::integral_constant<int, CMX_OUT_BF16>{}, u32x4{}) : f(std::integral_constant<int, CMX_OUT_BF16>{}, uint16_t{});
}

int check_routes(uint32_t tokens, uint32_t top_k, uint32_t rows) {
    CMX_REQUIRE(top_k >= 1 && top_k <= kMostRoutes, "top_k must be in [1, 64]");
    CMX_REQUIRE((uint64_t)tokens * top_k < (1ull << 31) && rows < (1u << 31), "tokens * top_k and rows must stay below 2^31");
    return CMX_OK;
}

}  // namespace
}  // namespace cmx

int cmx::preload_permute_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::moe_permute_kernel<u32x4>)));
    return CMX_OK;
}

extern "C" int cmx_moe_token_permute(const void* x, uint32_t ld_x, const int32_t* src2sorted, void* out, uint32_t ld_out, uint32_t rows, uint32_t tokens,
                                     uint32_t hidden, uint32_t top_k, uint32_t element_bytes, int zero_rest, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(element_bytes == 1 || element_bytes == 2 || element_bytes == 4, "elements of 1, 2 or 4 bytes");
    if (int rc = check_routes(tokens, top_k, rows); rc != CMX_OK) return rc;
    if (rows == 0 || hidden == 0 || (tokens == 0 && !zero_rest)) return CMX_OK;
    CMX_REQUIRE(out && (tokens == 0 || (x && src2sorted)), "null pointer");
    CMX_REQUIRE(ld_x >= hidden && ld_out >= hidden, "row pitch smaller than a row");
    const uint64_t xa = reinterpret_cast<uintptr_t>(x), oa = reinterpret_cast<uintptr_t>(out), row = (uint64_t)hidden * element_bytes;
    CMX_REQUIRE(xa % element_bytes == 0 && oa % element_bytes == 0, "pointers must be aligned to their elements");
    PermuteArgs p{};
    p.x = static_cast<const uint8_t*>(x);
    p.src2sorted = src2sorted;
    p.out = static_cast<uint8_t*>(out);
    p.ld_x = (size_t)ld_x * element_bytes;
    p.ld_out = (size_t)ld_out * element_bytes;
    p.tokens = tokens;
    p.top_k = top_k;
    p.rows = rows;
    if (zero_rest) p.clear = clear_job(rows, tokens * top_k);
    const uint32_t bytes = piece_bytes(row, {xa, oa, p.ld_x, p.ld_out});
    CMX_REQUIRE(row / bytes < (1ull << 32), "rows too long");
    p.vecs = (uint32_t)(row / bytes);
    const uint64_t blocks = p.clear.blocks + ((uint64_t)tokens * p.vecs + kThreads - 1) / kThreads;
    CMX_REQUIRE(fits_grid(blocks, kThreads), "too many elements");
    const auto kfn = bytes == 16 ? moe_permute_kernel<u32x4> : bytes == 8 ? moe_permute_kernel<u32x2> : bytes == 4 ? moe_permute_kernel<uint32_t>
                     : bytes == 2 ? moe_permute_kernel<uint16_t> : moe_permute_kernel<uint8_t>;
    hipLaunchKernelGGL(kfn, dim3((uint32_t)blocks), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}

extern "C" int cmx_moe_token_permute_grad(const void* dy, uint32_t ld_dy, uint32_t rows, const int32_t* src2sorted, void* dx, uint32_t ld_dx, uint32_t tokens,
                                          uint32_t hidden, uint32_t top_k, int type, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(type == CMX_OUT_BF16 || type == CMX_OUT_FP16 || type == CMX_OUT_FP32, "unknown type");
    if (int rc = check_routes(tokens, top_k, rows); rc != CMX_OK) return rc;
    if (tokens == 0 || hidden == 0) return CMX_OK;
    CMX_REQUIRE((dy || rows == 0) && src2sorted && dx, "null pointer");
    CMX_REQUIRE(ld_dy >= hidden && ld_dx >= hidden, "row pitch smaller than a row");
    const uint32_t size = type == CMX_OUT_FP32 ? 4 : 2;
    const uint64_t ya = reinterpret_cast<uintptr_t>(dy), xa = reinterpret_cast<uintptr_t>(dx);
    CMX_REQUIRE(ya % size == 0 && xa % size == 0, "pointers must be aligned to their elements");
    PermuteArgs p{};
    p.x = static_cast<const uint8_t*>(dy);
    p.src2sorted = src2sorted;
    p.out = static_cast<uint8_t*>(dx);
    p.ld_x = (size_t)ld_dy * size;
    p.ld_out = (size_t)ld_dx * size;
    p.tokens = tokens;
    p.top_k = top_k;
    p.rows = rows;
    p.vecs = hidden;
    return by_type(type, piece_bytes((uint64_t)hidden * size, {ya, xa, p.ld_x, p.ld_out}), [&](auto t, auto v) {
        return launch_permute_grad<decltype(t)::value, decltype(v)>(p, static_cast<hipStream_t>(stream));
    });
}

extern "C" int cmx_moe_token_unpermute_grad(const void* dout, uint32_t ld_dout, const void* y, uint32_t ld_y, uint32_t rows, const int32_t* src2sorted,
                                            const float* probs, void* dy, uint32_t ld_dy, float* dprobs, uint32_t tokens, uint32_t hidden, uint32_t top_k,
                                            int type, int zero_rest, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(type == CMX_OUT_BF16 || type == CMX_OUT_FP16 || type == CMX_OUT_FP32, "unknown type");
    if (int rc = check_routes(tokens, top_k, rows); rc != CMX_OK) return rc;
    if (tokens == 0 && (rows == 0 || hidden == 0 || !zero_rest)) return CMX_OK;
    CMX_REQUIRE((dy || rows == 0 || hidden == 0) && (tokens == 0 || (dout && src2sorted && probs && dprobs && (y || rows == 0))), "null pointer");
    CMX_REQUIRE(ld_dout >= hidden && ld_y >= hidden && ld_dy >= hidden, "row pitch smaller than a row");
    const uint32_t size = type == CMX_OUT_FP32 ? 4 : 2;
    const uint64_t ga = reinterpret_cast<uintptr_t>(dout), ya = reinterpret_cast<uintptr_t>(y), da = reinterpret_cast<uintptr_t>(dy);
    CMX_REQUIRE(ga % size == 0 && ya % size == 0 && da % size == 0, "pointers must be aligned to their elements");
    PermuteArgs p{};
    p.x = static_cast<const uint8_t*>(y);
    p.dout = static_cast<const uint8_t*>(dout);
    p.src2sorted = src2sorted;
    p.probs = probs;
    p.out = static_cast<uint8_t*>(dy);
    p.dprobs = dprobs;
    p.ld_x = (size_t)ld_y * size;
    p.ld_dout = (size_t)ld_dout * size;
    p.ld_out = (size_t)ld_dy * size;
    p.tokens = tokens;
    p.top_k = top_k;
    p.rows = rows;
    p.vecs = hidden;
    if (zero_rest && rows != 0 && hidden != 0) p.clear = clear_job(rows, tokens * top_k);
    return by_type(type, piece_bytes((uint64_t)hidden * size, {ga, ya, da, p.ld_x, p.ld_dout, p.ld_out}), [&](auto t, auto v) {
        return launch_unpermute_grad<decltype(t)::value, decltype(v)>(p, static_cast<hipStream_t>(stream));
    });
}
