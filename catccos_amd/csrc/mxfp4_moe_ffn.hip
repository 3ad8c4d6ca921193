// The routed FFN of a few tokens on MXFP4 expert weights, activations as they are (W4A16):
//
//   a[t, e] = p[t, e] * silu(x[t] . W1g[e]^T) * (x[t] . W1u[e]^T),   out[t] = sum over e of a[t, e] . W2[e]^T
//
// Two launches.  At decode an expert has one row or a few, so the time is that of reading the chosen experts' weights once: nothing is sorted or
// scattered beforehand.  A workgroup of the first kernel stands for one route and goes on only if that route is the first of its expert; then it collects the
// others, which become the columns of its matrix instructions.  a is kept as two bf16 halves whose sum carries 16 bits, so that out is
// rounded once.  The second kernel's workgroups own rows of W2 for all experts, so that a token's sum over its experts never leaves the workgroup; it
// is taken in an order that depends on the routing alone.
#include "mxfp4_rows.h"

namespace cmx {
namespace {

constexpr uint32_t kTokens = 64;         // of one pass over the weights; more tokens are taken in several
constexpr uint32_t kMaxTopK = 64;
constexpr uint32_t kUpWaves = 8, kDownWaves = 8;

struct FfnArgs {
    const uint8_t* x;                    // bf16 [m, k]
    const int32_t* idx;
    const float* gate;
    const uint8_t *w1, *w1_scale, *w2, *w2_scale;
    uint8_t* out;                        // bf16 [m, k]
    uint8_t* act;                        // two planes of bf16 [m * top_k, half]; only rows of a route that is the first of its token and expert
    size_t plane;                        // bytes
    uint32_t* counts;                    // [m * top_k]: routes of the expert whose first route this is in its pass, 0 elsewhere
    uint16_t* members;                   // [m * top_k, kTokens]: those routes, counted from the pass's first
    uint32_t m, k, half, experts, top_k;
};

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

__global__ __launch_bounds__(64 * kUpWaves) void mxfp4_moe_up_kernel(const FfnArgs a) {
    __shared__ v4f sums[kUpWaves][2][64];
    __shared__ uint16_t members[kTokens];
    __shared__ float weights[kTokens];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t token0 = blockIdx.z * kTokens, tokens = min(a.m - token0, kTokens), routes = tokens * a.top_k, first = blockIdx.y;
    if (first >= routes) return;
    const size_t route0 = (size_t)token0 * a.top_k;
    const int32_t* const idx = a.idx + route0;
    const int32_t e = idx[first];
    // every wavefront looks through the routes: the same answer in each
    uint32_t count = 0;
    bool leads = e >= 0 && (uint32_t)e < a.experts;
    for (uint32_t r0 = 0; leads && r0 < routes; r0 += 64) {
        const uint32_t r = r0 + lane;
        bool match = r < routes && idx[r] == e;
        if (__ballot(match && r < first)) leads = false;
        const uint32_t token = r / a.top_k;
        float p = 0.0f;
        if (match) {                                                  // an expert named twice by a token counts once, with both weights
            for (uint32_t s = token * a.top_k; s < r; ++s) match &= idx[s] != e;
            for (uint32_t s = r; s < (token + 1) * a.top_k; ++s) p += idx[s] == e ? a.gate[route0 + s] : 0.0f;
        }
        const uint64_t all = __ballot(match);
        if (match && wave == 0) {
            const uint32_t at = count + __popcll(all & ((1ull << lane) - 1));
            members[at] = (uint16_t)r;
            weights[at] = p;
        }
        count += __popcll(all);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.counts[route0 + first] = leads ? count : 0;
    if (!leads) return;
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x < count) a.members[(route0 + first) * kTokens + threadIdx.x] = members[threadIdx.x];

    const uint32_t blocks = a.k / 32, scale_pitch = (blocks + 1) & ~1u, tile = blockIdx.x * 16;
    RowsTile<kXBf16, 2, 1, 1> t;                                      // gate rows and their up rows
    t.blocks = blocks;
    t.plane = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const size_t row = (size_t)e * (2 * a.half) + i * a.half + tile + (lane & 15);
        t.a[i] = a.w1 + row * (a.k / 2) + (lane >> 4) * 16;
        t.scale[i] = a.w1_scale + row * scale_pitch + (lane >> 4);
    }
    for (uint32_t c0 = 0; c0 < count; c0 += 16) {
        const uint32_t c = min(c0 + (lane & 15), count - 1);          // (columns past the last repeat it, and are not stored)
        t.x[0] = a.x + ((size_t)(token0 + members[c] / a.top_k) * a.k + (lane >> 4) * 32) * 2;
        t.clear();
        t.run(wave, (blocks + 3) / 4, kUpWaves);
        if (c0) __syncthreads();
        sums[wave][0][lane] = t.acc[0][0];
        sums[wave][1][lane] = t.acc[1][0];
        __syncthreads();
        if (threadIdx.x < 256) {
            const uint32_t l = threadIdx.x >> 2, i = threadIdx.x & 3, col = c0 + (l & 15);
            float g = 0.0f, u = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kUpWaves; ++w) {
                g += sums[w][0][l][i];
                u += sums[w][1][l][i];
            }
            if (col < count) {
                const float v = weights[col] * (silu(g) * u), lead = __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
                const size_t at = ((route0 + members[col]) * a.half + tile + (l >> 4) * 4 + i) * 2;
                *reinterpret_cast<uint16_t*>(a.act + at) = (uint16_t)(__float_as_uint(v) >> 16);
                *reinterpret_cast<uint16_t*>(a.act + a.plane + at) = (uint16_t)f32_to_bf16(lead == v ? 0.0f : v - lead);
            }
        }
    }
}

__global__ __launch_bounds__(64 * kDownWaves) void mxfp4_moe_down_kernel(const FfnArgs a) {
    extern __shared__ float sums[];                                   // [wavefront][token][16 rows]
    __shared__ uint16_t leaders[kTokens * kMaxTopK];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = blockIdx.x * 16;
    const uint32_t token0 = blockIdx.y * kTokens, tokens = min(a.m - token0, kTokens), routes = tokens * a.top_k;
    const size_t route0 = (size_t)token0 * a.top_k;
    uint32_t experts = 0;
    for (uint32_t r0 = 0; r0 < routes; r0 += 64) {
        const bool leads = r0 + lane < routes && a.counts[route0 + r0 + lane] != 0;
        const uint64_t all = __ballot(leads);
        if (leads && wave == 0) leaders[experts + __popcll(all & ((1ull << lane) - 1))] = (uint16_t)(r0 + lane);
        experts += __popcll(all);
    }
    for (uint32_t i = threadIdx.x; i < kDownWaves * tokens * 16; i += blockDim.x) sums[i] = 0.0f;
    __syncthreads();

    const uint32_t blocks = a.half / 32, scale_pitch = (blocks + 1) & ~1u, units = (blocks + 3) / 4;
    uint32_t parts = 1;                                               // of an expert's K, where there are fewer experts than wavefronts
    while (experts * parts < kDownWaves && parts < units) parts *= 2;
    RowsTile<kXPlanes, 1, 1, 1> t;
    t.blocks = blocks;
    t.plane = a.plane;
    float* const mine = sums + (size_t)wave * tokens * 16;
    for (uint32_t item = wave; item < experts * parts; item += kDownWaves) {
        const uint32_t leader = leaders[item / parts], part = item % parts;
        const size_t route = route0 + leader;
        const uint32_t count = a.counts[route];
        const size_t row = (size_t)a.idx[route] * a.k + tile + (lane & 15);
        t.a[0] = a.w2 + row * (a.half / 2) + (lane >> 4) * 16;
        t.scale[0] = a.w2_scale + row * scale_pitch + (lane >> 4);
        for (uint32_t c0 = 0; c0 < count; c0 += 16) {
            const uint32_t c = c0 + (lane & 15), member = a.members[route * kTokens + min(c, count - 1)];
            t.x[0] = a.act + ((route0 + member) * a.half + (lane >> 4) * 32) * 2;
            t.clear();
            t.run(units * part / parts, units * (part + 1) / parts, 1);
            if (c < count) {                                          // the columns are different tokens
                v4f* const at = reinterpret_cast<v4f*>(mine + (member / a.top_k) * 16 + (lane >> 4) * 4);
                *at += t.acc[0][0];
            }
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < tokens * 4; i += blockDim.x) {
        v4f v = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t w = 0; w < kDownWaves; ++w) v += reinterpret_cast<const v4f*>(sums)[w * tokens * 4 + i];
        const uint32_t packed[2] = {cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])};
        __builtin_memcpy(a.out + ((size_t)(token0 + i / 4) * a.k + tile + (i & 3) * 4) * 2, packed, 8);
    }
}

// the workspace: planes, counts, members
struct FfnLayout {
    size_t counts, members, plane, total;
};
FfnLayout ffn_layout(uint64_t m, uint64_t n, uint64_t top_k) {
    FfnLayout l;
    const size_t routes = (size_t)m * top_k;
    l.plane = round_up_sz(routes * (n / 2) * 2, 256);
    l.counts = 2 * l.plane;
    l.members = l.counts + round_up_sz(routes * 4, 256);
    l.total = l.members + round_up_sz(routes * kTokens * 2, 256);
    return l;
}

}  // namespace
}  // namespace cmx

int cmx::preload_moe_ffn_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::mxfp4_moe_up_kernel)));
    return CMX_OK;
}

extern "C" size_t cmx_mxfp4_moe_ffn_workspace_bytes(uint32_t m, uint32_t n, uint32_t top_k) { return cmx::ffn_layout(m, n, top_k).total; }

extern "C" int cmx_mxfp4_moe_ffn(const void* x, const int32_t* expert_idx, const float* gate_weight, const uint8_t* w1, const uint8_t* w1_scale,
                                 const uint8_t* w2, const uint8_t* w2_scale, void* out, uint8_t* workspace, uint32_t m, uint32_t k, uint32_t n,
                                 uint32_t experts, uint32_t top_k, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(k > 0 && k % 32 == 0, "k must be a positive multiple of 32");
    CMX_REQUIRE(n > 0 && n % 64 == 0, "n must be a positive multiple of 64");
    CMX_REQUIRE(experts > 0 && experts < (1u << 31), "experts must be in [1, 2^31)");
    CMX_REQUIRE(top_k > 0 && top_k <= kMaxTopK, "top_k must be in [1, 64]");
    CMX_REQUIRE((uint64_t)m * top_k < (1ull << 31) && m <= 65535u * kTokens, "too many tokens");
    if (m == 0) return CMX_OK;
    CMX_REQUIRE(x && expert_idx && gate_weight && w1 && w1_scale && w2 && w2_scale && out && workspace, "null pointer");
    CMX_REQUIRE(aligned16(w1) && aligned16(w2), "weights must be 16-byte aligned");
    CMX_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "workspace must be 256-byte aligned");
    CMX_REQUIRE(((reinterpret_cast<uintptr_t>(expert_idx) | reinterpret_cast<uintptr_t>(gate_weight)) & 3u) == 0 &&
                ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 1u) == 0, "pointers must be aligned to their elements");
    const FfnLayout l = ffn_layout(m, n, top_k);
    const FfnArgs a = {static_cast<const uint8_t*>(x), expert_idx, gate_weight, w1, w1_scale, w2, w2_scale, static_cast<uint8_t*>(out), workspace, l.plane,
                       reinterpret_cast<uint32_t*>(workspace + l.counts), reinterpret_cast<uint16_t*>(workspace + l.members), m, k, n / 2, experts, top_k};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t passes = ceil_div(m, kTokens), tokens = m < kTokens ? m : kTokens;
    hipLaunchKernelGGL(mxfp4_moe_up_kernel, dim3(n / 32, tokens * top_k, passes), dim3(64 * kUpWaves), 0, s, a);
    CMX_LAUNCH_CHECK();
    hipLaunchKernelGGL(mxfp4_moe_down_kernel, dim3(k / 16, passes), dim3(64 * kDownWaves), kDownWaves * tokens * 16 * 4, s, a);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}
