// The routed FFN of a few tokens on MXFP4 expert weights, activations as they are (W4A16):
//
//   a[t, e] = p[t, e] * silu(x[t] . W1g[e]^T) * (x[t] . W1u[e]^T),   out[t] = sum over e of a[t, e] . W2[e]^T
//
// Two launches.  At decode an expert has one row or a few, so the time is that of reading the chosen experts' weights once: nothing is sorted or
// scattered beforehand.  A workgroup of the first kernel stands for one route and goes on only if that route is the first of its expert; then it collects the
// others, which become the columns of its matrix instructions.  a is kept as two bf16 halves whose sum carries 16 bits, so that out is
// rounded once.  The second kernel's workgroups own rows of W2 for all experts, so that a token's sum over its experts never leaves the workgroup; it
// is taken in an order that depends on the routing alone.
#include "mx_launch.h"
#include "mxfp4_rows.h"

#ifndef CMX_UPW
#define CMX_UPW 2048
#endif
namespace cmx {
namespace {

constexpr uint32_t kTokens = 64;         // of one pass over the weights; more tokens are taken in several
constexpr uint32_t kMaxTopK = 64;
constexpr uint32_t kUpWaves = 8, kDownWaves = 8;
constexpr uint32_t kMaxLds = 150 * 1024; // besides the lists

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
    uint32_t up_columns, down_columns;   // routes of an expert that one reading of its weights serves
    uint32_t up_parts;                   // of K: wavefronts of a workgroup that share a row tile of the first matmul
};

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

__global__ __launch_bounds__(64 * kUpWaves, 4) void mxfp4_moe_up_kernel(const FfnArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // activations of each wavefront, then sums: [wavefront][gate, up][lane]
    __shared__ uint16_t members[kTokens];
    __shared__ float weights[kTokens];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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

    const uint32_t blocks = a.k / 32, scale_pitch = (blocks + 1) & ~1u, part = wave % a.up_parts;
    const uint32_t tile = (blockIdx.x * (kUpWaves / a.up_parts) + wave / a.up_parts) * 16;
    const bool works = tile < a.half;                                 // (the last workgroup of an expert may have wavefronts to spare)
    RowsTile<kXBf16, 2> t;                                            // gate rows and their up rows
    t.blocks = blocks;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const size_t row = (size_t)e * (2 * a.half) + i * a.half + (works ? tile : 0) + (lane & 15);
        t.a[i] = a.w1 + row * (a.k / 2) + (lane >> 4) * 16;
        t.scale[i] = a.w1_scale + row * scale_pitch;
    }
    XColumns<kXBf16, true> x;
    x.x = a.x + (size_t)token0 * a.k * 2;
    x.pitch = (size_t)a.k * 2;
    x.plane = 0;
    x.row_bytes = a.k * 2;
    x.lds = lds + wave * a.up_columns * XTraits<kXBf16>::kPitch;
    v4f(*const sums)[2][64] = reinterpret_cast<v4f(*)[2][64]>(lds);
    for (uint32_t c0 = 0; c0 < count; c0 += a.up_columns) {
        x.columns = min(count - c0, a.up_columns);
        x.row = members[c0 + min(lane, x.columns - 1)] / a.top_k;
        t.clear();
        if (works) t.run(x, part, (blocks + kUnitBlocks - 1) / kUnitBlocks, a.up_parts);
        if (a.up_parts > 1) {
            __syncthreads();
            if (part != 0) {
                sums[wave][0][lane] = t.acc[0];
                sums[wave][1][lane] = t.acc[1];
            }
            __syncthreads();
            if (part == 0) {
                for (uint32_t w = 1; w < a.up_parts; ++w) {
                    t.acc[0] += sums[wave + w][0][lane];
                    t.acc[1] += sums[wave + w][1][lane];
                }
            }
            if (c0 + a.up_columns < count) __syncthreads();           // (the next activations go where these sums are)
        }
        const uint32_t c = lane & 15;
        if (part == 0 && works && c < x.columns) {
            uint32_t lead[2], rest[2];
            float v[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = weights[c0 + c] * (silu(t.acc[0][i]) * t.acc[1][i]);
                const float high = __uint_as_float(__float_as_uint(v[i]) & 0xFFFF0000u);
                w[i] = high == v[i] ? 0.0f : v[i] - high;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                lead[i] = __builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);
                rest[i] = cvt_pk_bf16(w[2 * i], w[2 * i + 1]);
            }
            const size_t at = ((route0 + members[c0 + c]) * a.half + tile + (lane >> 4) * 4) * 2;
            __builtin_memcpy(a.act + at, lead, 8);
            __builtin_memcpy(a.act + a.plane + at, rest, 8);
        }
    }
}

__global__ __launch_bounds__(64 * kDownWaves, 4) void mxfp4_moe_down_kernel(const FfnArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // activations of each wavefront; sums: [wavefront][token][16 rows]
    __shared__ uint16_t leaders[kTokens * kMaxTopK];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tile = blockIdx.x * 16;
    const uint32_t token0 = blockIdx.y * kTokens, tokens = min(a.m - token0, kTokens), routes = tokens * a.top_k;
    const size_t route0 = (size_t)token0 * a.top_k;
    uint32_t experts = 0;
    for (uint32_t r0 = 0; r0 < routes; r0 += 64) {
        const bool leads = r0 + lane < routes && a.counts[route0 + r0 + lane] != 0;
        const uint64_t all = __ballot(leads);
        if (leads && wave == 0) leaders[experts + __popcll(all & ((1ull << lane) - 1))] = (uint16_t)(r0 + lane);
        experts += __popcll(all);
    }
    const uint32_t staging = a.down_columns * XTraits<kXPlanes>::kPitch;
    float* const sums = reinterpret_cast<float*>(lds + kDownWaves * staging);
    for (uint32_t i = threadIdx.x; i < kDownWaves * tokens * 16; i += blockDim.x) sums[i] = 0.0f;
    __syncthreads();

    const uint32_t blocks = a.half / 32, scale_pitch = (blocks + 1) & ~1u, units = (blocks + kUnitBlocks - 1) / kUnitBlocks;
    uint32_t parts = 1;                                               // of an expert's K, where there are fewer experts than wavefronts
    while (experts * parts < kDownWaves && parts < units) parts *= 2;
    RowsTile<kXPlanes, 1> t;
    t.blocks = blocks;
    XColumns<kXPlanes, true> x;
    x.x = a.act + route0 * a.half * 2;
    x.pitch = (size_t)a.half * 2;
    x.plane = a.plane;
    x.row_bytes = a.half * 2;
    x.lds = lds + wave * staging;
    float* const mine = sums + (size_t)wave * tokens * 16;
    for (uint32_t item = wave; item < experts * parts; item += kDownWaves) {
        const uint32_t leader = leaders[item / parts], part = item % parts;
        const size_t route = route0 + leader;
        const uint32_t count = a.counts[route];
        const size_t row = (size_t)a.idx[route] * a.k + tile + (lane & 15);
        t.a[0] = a.w2 + row * (a.half / 2) + (lane >> 4) * 16;
        t.scale[0] = a.w2_scale + row * scale_pitch;
        for (uint32_t c0 = 0; c0 < count; c0 += a.down_columns) {
            x.columns = min(count - c0, a.down_columns);
            const uint32_t c = lane & 15, member = a.members[route * kTokens + c0 + min(c, x.columns - 1)];
            x.row = member;
            t.clear();
            t.run(x, units * part / parts, units * (part + 1) / parts, 1);
            if (c < x.columns) {                                      // the columns are different tokens
                v4f* const at = reinterpret_cast<v4f*>(mine + (member / a.top_k) * 16 + (lane >> 4) * 4);
                *at += t.acc[0];
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
                (reinterpret_cast<uintptr_t>(out) & 1u) == 0, "pointers must be aligned to their elements");
    CMX_REQUIRE(aligned16(x), "x must be 16-byte aligned");
    const FfnLayout l = ffn_layout(m, n, top_k);
    FfnArgs a = {static_cast<const uint8_t*>(x), expert_idx, gate_weight, w1, w1_scale, w2, w2_scale, static_cast<uint8_t*>(out), workspace, l.plane,
                       reinterpret_cast<uint32_t*>(workspace + l.counts), reinterpret_cast<uint16_t*>(workspace + l.members), m, k, n / 2, experts, top_k, 0, 0, 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t passes = ceil_div(m, kTokens), tokens = m < kTokens ? m : kTokens;
    a.up_columns = (uint64_t)tokens * top_k > 2ull * experts ? 16 : 4;
    a.up_columns = tokens < a.up_columns ? tokens : a.up_columns;
    a.down_columns = tokens < 4 ? tokens : 4;
    // K is shared out where the row tiles of all experts alone would leave the card without enough wavefronts
    const uint64_t tiles = (uint64_t)(tokens * top_k < experts ? tokens * top_k : experts) * (n / 32);
    const uint32_t units = ceil_div(k, kUnitK);
    a.up_parts = 1;
    while (a.up_parts < kUpWaves && a.up_parts * 2 <= units && tiles * a.up_parts < CMX_UPW) a.up_parts *= 2;
    if (int rc = allow_dynamic_lds<mxfp4_moe_up_kernel, kMaxLds>(); rc != CMX_OK) return rc;
    if (int rc = allow_dynamic_lds<mxfp4_moe_down_kernel, kMaxLds>(); rc != CMX_OK) return rc;
    const uint32_t up_each = a.up_columns * XTraits<kXBf16>::kPitch;
    hipLaunchKernelGGL(mxfp4_moe_up_kernel, dim3(ceil_div(n / 32, kUpWaves / a.up_parts), tokens * top_k, passes), dim3(64 * kUpWaves), kUpWaves * (up_each > 2048 ? up_each : 2048), s, a);
    CMX_LAUNCH_CHECK();
    hipLaunchKernelGGL(mxfp4_moe_down_kernel, dim3(k / 16, passes), dim3(64 * kDownWaves),
                       kDownWaves * (a.down_columns * XTraits<kXPlanes>::kPitch + tokens * 64), s, a);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}
