// The routed FFN of a few tokens on MXFP4 expert weights, activations as they are (W4A16):
//
//   a[t, e] = p[t, e] * silu(x[t] . W1g[e]^T) * (x[t] . W1u[e]^T),   out[t] = sum over e of a[t, e] . W2[e]^T
//
// Two launches.  At decode an expert has one row or a few, so the time is that of reading the chosen experts' weights once: nothing is sorted or
// scattered beforehand.  A workgroup of the first kernel stands for an expert or, where experts outnumber routes, for one route, and goes on only if that
// is the first of its expert; it collects the expert's routes, which become the columns of its matrix instructions.  a is kept as two bf16 halves whose sum carries 16 bits, so that out is
// rounded once.  The second kernel's workgroups own rows of W2 for all experts, so that a token's sum over its experts never leaves the workgroup; it
// is taken in an order that depends on the routing alone.
//
// Bound by the weights of the experts that are named.  Measured, k = 7168, n = 4096, 8 of 256 experts a token: one token 24 + 16 us (187 MB, 4.6 TB/s), 32
// tokens 715 to 740 us (3.8 GB, 5.2 TB/s), of which the first takes 445.
#include "mx_launch.h"
#include "mxfp4_rows.h"

namespace cmx {
namespace {

constexpr uint32_t kTokens = 64;         // of one pass over the weights; more tokens are taken in several
constexpr uint32_t kMaxTopK = 64, kNone = ~0u;
constexpr uint32_t kMaxLds = 159 * 1024;
// First matmul, by the columns of a wavefront: small workgroups, three of which share a CU, so that one works while another starts or ends (32 tokens, 256
// experts: 445 us; one of eight wavefronts 514; one token 24 us and 35); with many columns LDS has room for one (45 tokens, 16 experts, K = 992: 11 us; of
// four wavefronts 16).
constexpr uint32_t up_waves(int columns) { return columns <= 4 ? 4 : 8; }
// Second matmul: as many as registers allow (45 tokens, 128 experts, k = 736: 36.6 us for both matmuls with 8, 35.0 with 12; 90 tokens, 64 experts, k = 576: 68.8 and
// 63.8).
constexpr uint32_t down_waves(int row_tiles, int columns) { return row_tiles == 1 && columns <= 4 ? 12 : 8; }
constexpr uint32_t kEnoughWaves = 1024;          // of the first matmul, below which K is shared out (45 tokens, 16 experts, K = 992: 11 us, unshared 13; one token, 8 experts,
                                                 // K = 7168, that has 1024: 24 us, shared further 28)

struct FfnArgs {
    const uint8_t* x;                    // bf16 [m, k]
    const int32_t* idx;
    const float* gate;
    const uint8_t *w1, *w1_scale, *w2, *w2_scale;
    uint8_t* out;                        // bf16 [m, k]
    uint8_t* act;                        // two planes of bf16 [m * top_k, half]; only rows of a route that is the first of its token and expert
    size_t plane;                        // bytes
    uint32_t* counts;                    // [m * top_k]: routes of the expert whose first route this is in its pass, 0 elsewhere
    uint32_t* places;                    // [m * top_k]: first route of the expert (counted in the pass) * kTokens + place among its routes, kNone
    uint32_t m, k, half, experts, top_k;
    uint32_t pass, down_pass;            // tokens of one pass of the two matmuls; a pass of the first holds whole ones of the second
    bool by_expert;                      // workgroups of the first matmul stand for experts, not for routes
    uint32_t up_parts;                   // of K: wavefronts of a workgroup that share a row tile of the first matmul
};

__device__ __forceinline__ uint32_t scalar(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

// COLUMNS: routes of an expert that one reading of its weights serves
template <int COLUMNS>
__global__ __launch_bounds__(64 * up_waves(COLUMNS), COLUMNS <= 4 ? 3 : 2) void mxfp4_moe_up_kernel(const FfnArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // a stage for each wavefront, then sums: [wavefront][gate, up][lane]
    __shared__ uint16_t members[kTokens];                             // the expert's routes, counted in the pass
    __shared__ float weights[kTokens];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t token0 = blockIdx.z * a.pass, tokens = min(a.m - token0, a.pass), routes = tokens * a.top_k;
    if (!a.by_expert && blockIdx.y >= routes) return;
    const size_t route0 = (size_t)token0 * a.top_k;
    int32_t* const idx = reinterpret_cast<int32_t*>(lds);             // of the pass, until the stages take the place: one wait for memory, not one a look
    for (uint32_t r = threadIdx.x; r < routes; r += blockDim.x) idx[r] = a.idx[route0 + r];
    __syncthreads();
    const uint32_t e = a.by_expert ? blockIdx.y : scalar((uint32_t)idx[blockIdx.y]);
    const bool tells = blockIdx.x == 0 && wave == 0;                  // (one wavefront writes down for the second kernel what all find out)
    // every wavefront looks through the routes: the same answer in each
    uint32_t count = 0, first = kNone;
    for (uint32_t r0 = 0; r0 < routes; r0 += 64) {
        const uint32_t r = r0 + lane, named = r < routes ? (uint32_t)idx[r] : e;
        if (tells && blockIdx.y == 0 && named >= a.experts && r < routes) {       // no expert: nobody else's either
            a.places[route0 + r] = kNone;
            a.counts[route0 + r] = 0;
        }
        const bool match = r < routes && named == e && e < a.experts;
        const uint64_t matches = __ballot(match);
        if (matches == 0) continue;
        if (first == kNone) first = r0 + (uint32_t)__builtin_ctzll(matches);
        if (!a.by_expert && first != blockIdx.y) return;
        const uint32_t token = r / a.top_k;
        float p = 0.0f;
        bool counted = match;
        if (match) {                                                  // an expert named twice by a token counts once, with both weights
            for (uint32_t s = token * a.top_k; s < r; ++s) counted &= (uint32_t)idx[s] != e;
            for (uint32_t s = r; s < (token + 1) * a.top_k; ++s) p += (uint32_t)idx[s] == e ? a.gate[route0 + s] : 0.0f;
        }
        const uint64_t all = __ballot(counted);
        const uint32_t at = count + __popcll(all & ((1ull << lane) - 1));
        if (counted && wave == 0) {
            members[at] = (uint16_t)r;
            weights[at] = p;
        }
        if (match && !counted && tells) {
            a.places[route0 + r] = kNone;
            a.counts[route0 + r] = 0;
        }
        count += __popcll(all);
    }
    if (count == 0) return;
    __syncthreads();
    if (tells && lane < count) {                                      // lane: place among the expert's routes (no more than tokens)
        const uint32_t r = members[lane], per = a.down_pass * a.top_k, pass = r / per;
        const uint64_t starts = __ballot(lane == 0 || members[max(lane, 1u) - 1] / per != pass);
        const uint32_t start = 63 - (uint32_t)__builtin_clzll(starts & (~0ull >> (63 - lane)));
        const uint64_t later = starts >> lane >> 1;
        a.places[route0 + r] = (members[start] - pass * per) * kTokens + lane - start;
        a.counts[route0 + r] = start != lane ? 0 : (later ? 1 + (uint32_t)__builtin_ctzll(later) : count - lane);
    }

    const uint32_t blocks = a.k / 32, scale_pitch = (blocks + 1) & ~1u, part = wave % a.up_parts;
    const uint32_t tile = (blockIdx.x * (waves / a.up_parts) + wave / a.up_parts) * 16;
    const bool works = tile < a.half;                                 // (the last workgroup of an expert may have wavefronts to spare)
    RowsStream<kXBf16, 2, COLUMNS, COLUMNS <= 4> t;                       // gate rows and their up rows
    t.blocks = blocks;
    const size_t w1_row = (size_t)e * (2 * a.half);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        t.set_rows(i, a.w1 + w1_row * (a.k / 2), a.k / 2, a.w1_scale + w1_row * scale_pitch, scale_pitch, i * a.half + (works ? tile : 0), 2 * a.half - 1);
    t.x = a.x + (size_t)token0 * a.k * 2;
    t.x_pitch = (size_t)a.k * 2;
    t.plane = 0;
    t.stage = lds_address(lds) + wave * kStageBytes<kXBf16, 2, COLUMNS>;
    v4f(*const sums)[2][64] = reinterpret_cast<v4f(*)[2][64]>(lds);
    for (uint32_t c0 = 0; c0 < count; c0 += COLUMNS) {
        const uint32_t columns = min(count - c0, (uint32_t)COLUMNS);
        t.row = members[c0 + min(lane, columns - 1)] / a.top_k;
        t.clear();
        if (works) t.run(part, (blocks + kUnitBlocks - 1) / kUnitBlocks, a.up_parts);
        if (a.up_parts > 1) {
            __syncthreads();
            if (part != 0) {
                sums[wave][0][lane] = t.sum(0);
                sums[wave][1][lane] = t.sum(1);
            }
            __syncthreads();
            if (part == 0) {
                for (uint32_t w = 1; w < a.up_parts; ++w) {
                    t.acc[0][0] += sums[wave + w][0][lane];
                    t.acc[1][0] += sums[wave + w][1][lane];
                }
            }
            if (c0 + COLUMNS < count) __syncthreads();           // (the next activations go where these sums are)
        }
        const uint32_t c = lane & 15;
        if (part == 0 && works && c < columns) {
            uint32_t lead[2], rest[2];
            float v[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = weights[c0 + c] * (silu(t.acc[0][0][i]) * t.acc[1][0][i]);
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

// RT x 16 rows of every W2
template <int RT, int COLUMNS>
__global__ __launch_bounds__(64 * down_waves(RT, COLUMNS)) void mxfp4_moe_down_kernel(const FfnArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];     // a stage for each wavefront; sums: [wavefront][token][RT * 16 rows]; lists
    __shared__ uint32_t experts_named;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t tile = blockIdx.x * (RT * 16);
    const uint32_t token0 = blockIdx.y * a.down_pass, tokens = min(a.m - token0, a.down_pass), routes = tokens * a.top_k;
    const size_t route0 = (size_t)token0 * a.top_k;
    float* const sums = reinterpret_cast<float*>(lds + waves * kStageBytes<kXPlanes, RT, COLUMNS>);
    // experts with a route in this pass, in the order of their first routes: expert, its number of routes, where they begin in `members`
    uint32_t* const expert_of = reinterpret_cast<uint32_t*>(sums + (size_t)waves * tokens * (RT * 16));
    uint16_t* const begin_of = reinterpret_cast<uint16_t*>(expert_of + routes);
    uint16_t* const begin_of_route = begin_of + routes + 1;           // by first route
    uint16_t* const members = begin_of_route + routes;
    const uint32_t place0 = threadIdx.x < routes ? a.places[route0 + threadIdx.x] : kNone;
    if (wave == 0) {
        uint32_t experts = 0, all_members = 0, count = lane < routes ? a.counts[route0 + lane] : 0;
        int32_t expert = lane < routes ? a.idx[route0 + lane] : 0;
        for (uint32_t r0 = 0; r0 < routes; r0 += 64) {
            const uint32_t r = r0 + lane, ahead = r + 64;
            const uint32_t next_count = ahead < routes ? a.counts[route0 + ahead] : 0;
            const int32_t next_expert = ahead < routes ? a.idx[route0 + ahead] : 0;
            const uint64_t leads = __ballot(count != 0);
            uint32_t before = count;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const uint32_t v = (uint32_t)__shfl_up((int)before, d);
                before += lane >= (uint32_t)d ? v : 0;
            }
            const uint32_t begin = all_members + before - count;
            if (count != 0) {
                const uint32_t at = experts + __popcll(leads & ((1ull << lane) - 1));
                expert_of[at] = (uint32_t)expert;
                begin_of[at] = (uint16_t)begin;
                begin_of_route[r] = (uint16_t)begin;
            }
            experts += __popcll(leads);
            all_members += (uint32_t)__builtin_amdgcn_readlane((int)before, 63);
            count = next_count;
            expert = next_expert;
        }
        if (lane == 0) {
            begin_of[experts] = (uint16_t)all_members;
            experts_named = experts;
        }
    }
    for (uint32_t i = threadIdx.x; i < waves * tokens * (RT * 4); i += blockDim.x) reinterpret_cast<v4f*>(sums)[i] = (v4f){0, 0, 0, 0};
    __syncthreads();
    for (uint32_t r = threadIdx.x; r < routes; r += blockDim.x) {
        const uint32_t place = r == threadIdx.x ? place0 : a.places[route0 + r];
        if (place != kNone) members[begin_of_route[place / kTokens] + place % kTokens] = (uint16_t)r;
    }
    __syncthreads();
    const uint32_t experts = scalar(experts_named);

    const uint32_t blocks = a.half / 32, scale_pitch = (blocks + 1) & ~1u, units = (blocks + kUnitBlocks - 1) / kUnitBlocks;
    uint32_t parts = 1;                                               // of an expert's K, where there are fewer experts than wavefronts
    while (experts * parts < waves && parts * 2 <= units) parts *= 2;
    RowsStream<kXPlanes, RT, COLUMNS, COLUMNS <= 4> t;
    t.blocks = blocks;
    t.x = a.act + route0 * a.half * 2;
    t.x_pitch = (size_t)a.half * 2;
    t.plane = a.plane;
    t.stage = lds_address(lds) + wave * kStageBytes<kXPlanes, RT, COLUMNS>;
    float* const mine = sums + (size_t)wave * tokens * (RT * 16);
    // A wavefront's work is a sequence of units: of its share of an expert's K for up to COLUMNS of its routes, then the next columns, then the next
    // expert.  The next one is requested before the current one is multiplied, across all these borders.
    struct Position {
        uint32_t item, begin, columns, unit, last;                    // columns: routes members[begin, begin + columns)
    };
    const auto enter = [&](Position& p) {                             // weights and columns of an item and its columns from p.begin on
        const uint32_t at = p.item / parts, part = p.item % parts;
        p.columns = min(scalar(begin_of[at + 1]) - p.begin, (uint32_t)COLUMNS);
        p.unit = units * part / parts;
        p.last = units * (part + 1) / parts;
        t.row = members[p.begin + min(lane & 15, p.columns - 1)];
        const size_t w2_row = (size_t)scalar(expert_of[at]) * a.k;
#pragma unroll
        for (int i = 0; i < RT; ++i)
            t.set_rows(i, a.w2 + w2_row * (a.half / 2), a.half / 2, a.w2_scale + w2_row * scale_pitch, scale_pitch, tile + i * 16, a.k - 1);
    };
    const uint32_t items = experts * parts;
    Position now = {wave, 0, 0, 0, 0};
    if (wave < items) {
        now.begin = scalar(begin_of[wave / parts]);
        enter(now);
        uint32_t member = t.row;                                      // (of this lane's column)
        typename RowsStream<kXPlanes, RT, COLUMNS, COLUMNS <= 4>::Unit u;
        t.load(u, now.unit);
        t.clear();
        while (true) {
            Position next = now;
            uint32_t next_member = member;
            bool more = true;
            t.turn(u, now.unit, [&](auto& v) {
                ++next.unit;
                if (next.unit == now.last) {
                    next.begin += now.columns;
                    if (next.begin == scalar(begin_of[now.item / parts + 1])) {
                        next.item += waves;
                        more = next.item < items;
                        if (more) next.begin = scalar(begin_of[next.item / parts]);
                    }
                    if (more) {
                        enter(next);
                        next_member = t.row;
                    }
                }
                if (more) t.load(v, next.unit);
            });
            if (now.unit + 1 == now.last) {
                if ((lane & 15) < now.columns) {                      // the columns are different tokens
                    v4f* const at = reinterpret_cast<v4f*>(mine + (member / a.top_k) * (RT * 16) + (lane >> 4) * 4);
#pragma unroll
                    for (int i = 0; i < RT; ++i) at[i * 4] += t.sum(i);
                }
                t.clear();
            }
            if (!more) break;
            now = next;
            member = next_member;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < tokens * (RT * 4); i += blockDim.x) {
        const uint32_t row = tile + i % (RT * 4) * 4;
        if (row >= a.k) continue;
        v4f v = {0, 0, 0, 0};
        for (uint32_t w = 0; w < waves; ++w) v += reinterpret_cast<const v4f*>(sums)[w * tokens * (RT * 4) + i];
        const uint32_t packed[2] = {cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])};
        __builtin_memcpy(a.out + ((size_t)(token0 + i / (RT * 4)) * a.k + row) * 2, packed, 8);
    }
}

// the workspace: planes, counts, places
struct FfnLayout {
    size_t counts, places, plane, total;
};
FfnLayout ffn_layout(uint64_t m, uint64_t n, uint64_t top_k) {
    FfnLayout l;
    const size_t routes = (size_t)m * top_k;
    l.plane = round_up_sz(routes * (n / 2) * 2, 256);
    l.counts = 2 * l.plane;
    l.places = l.counts + round_up_sz(routes * 4, 256);
    l.total = l.places + round_up_sz(routes * 4, 256);
    return l;
}

}  // namespace
}  // namespace cmx

int cmx::preload_moe_ffn_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::mxfp4_moe_up_kernel<1>)));
    return CMX_OK;
}

extern "C" size_t cmx_mxfp4_moe_ffn_workspace_bytes(uint32_t m, uint32_t n, uint32_t top_k) { return cmx::ffn_layout(m, n, top_k).total; }

extern "C" int cmx_mxfp4_moe_ffn(const void* x, const int32_t* expert_idx, const float* gate_weight, const uint8_t* w1, const uint8_t* w1_scale,
                                 const uint8_t* w2, const uint8_t* w2_scale, void* out, uint8_t* workspace, uint32_t m, uint32_t k, uint32_t n,
                                 uint32_t experts, uint32_t top_k, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(k > 0 && k % 32 == 0 && k <= (1u << 26), "k must be a positive multiple of 32, at most 2^26");
    CMX_REQUIRE(n > 0 && n % 64 == 0 && n <= (1u << 26), "n must be a positive multiple of 64, at most 2^26");
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
                       reinterpret_cast<uint32_t*>(workspace + l.counts), reinterpret_cast<uint32_t*>(workspace + l.places), m, k, n / 2, experts, top_k, 0, 0, false, 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    int cus;
    if (int rc = cu_count(&cus); rc != CMX_OK) return rc;
    // The second matmul's workgroups are few where k is small: then its tokens are spread over more of them, as long as there are CUs for all (12 tokens, 256
    // experts, k = 352: 42 us for both matmuls with one pass, 21 with six; 61 tokens, 8 experts, k = 512: 58 with four passes, 46 with eight).
    a.down_pass = ceil_div(m, ceil_div(m, kTokens));
    uint32_t halved = 0;
    while (a.down_pass > 1 && (uint64_t)ceil_div(k, 16) * ceil_div(m, ceil_div(a.down_pass, 2)) <= (uint32_t)cus) {
        a.down_pass = ceil_div(a.down_pass, 2);
        ++halved;
    }
    a.pass = a.down_pass << halved;
    const uint32_t passes = ceil_div(m, a.pass), tokens = a.pass, most = tokens * top_k;
    // (a workgroup that stands for no expert or for another's is started and ended for nothing; 45 tokens of 3 routes, 16 experts: 17.6 us by route, 10.8 by expert)
    a.by_expert = experts <= most;
    // K is shared out where the row tiles of all experts alone would leave the card without enough wavefronts
    const uint64_t tiles = (uint64_t)(most < experts ? most : experts) * (n / 32);
    const uint32_t units = ceil_div(k, kUnitK);
    const auto up = [&](auto c) -> int {
        constexpr uint32_t kEach = kStageBytes<kXBf16, 2, c.value>, kFit = kMaxLds / kEach, kWaves = kFit < up_waves(c.value) ? kFit : up_waves(c.value);
        static_assert(kWaves >= 4 && 4 * kEach >= kTokens * kMaxTopK * 4, "the pass's routes fit where the stages are");
        if (int rc = allow_dynamic_lds<mxfp4_moe_up_kernel<c.value>, kWaves * kEach>(); rc != CMX_OK) return rc;
        a.up_parts = 1;
        while (a.up_parts * 2 <= kWaves && a.up_parts * 2 <= units && tiles * a.up_parts < kEnoughWaves) a.up_parts *= 2;
        const uint32_t waves = kWaves - kWaves % a.up_parts;
        hipLaunchKernelGGL((mxfp4_moe_up_kernel<c.value>), dim3(ceil_div(n / 32, waves / a.up_parts), a.by_expert ? experts : most, passes), dim3(64 * waves), waves * kEach, s, a);
        CMX_LAUNCH_CHECK();
        return CMX_OK;
    };
    const uint32_t down_most = a.down_pass * top_k;
    const auto down = [&](auto rt, auto c) -> int {
        const uint32_t each = kStageBytes<kXPlanes, rt.value, c.value> + a.down_pass * 64 * rt.value, lists = down_most * 10 + 16;
        const uint32_t fit = (kMaxLds - lists) / each, most_waves = down_waves(rt.value, c.value), waves = fit < most_waves ? fit : most_waves;
        if (int rc = allow_dynamic_lds<mxfp4_moe_down_kernel<rt.value, c.value>, kMaxLds>(); rc != CMX_OK) return rc;
        hipLaunchKernelGGL((mxfp4_moe_down_kernel<rt.value, c.value>), dim3(ceil_div(k, 16 * rt.value), ceil_div(m, a.down_pass)), dim3(64 * waves), waves * each + lists, s, a);
        CMX_LAUNCH_CHECK();
        return CMX_OK;
    };
    // Columns: as many routes as most experts have; what the others have more costs another reading of their weights, and columns that stand empty cost
    // wavefronts.  Routes spread at random, one for each of 256 experts on average: 88 % of those that have any have at most two and 97 % three.  (90 tokens of 3
    // routes, 64 experts: 74 us with 16 columns in the first matmul, 63 with 8; 64 tokens of 6, 64 experts, in two passes: 103 us with 8 columns in the
    // second, 95 with 4; 28 tokens of 3, 16 experts, one pass: 40 and 45.)
    const auto per_expert = [&](uint32_t routes, uint32_t by) { return routes <= (uint64_t)by * experts; };
    const uint32_t up_columns = per_expert(most, 2) && tokens > 3 ? 3 : (per_expert(most, 5) && tokens > 8 ? 8 : tokens);
    int rc;
    if (up_columns <= 1) rc = up(std::integral_constant<int, 1>());
    else if (up_columns <= 3) rc = up(std::integral_constant<int, 3>());
    else if (up_columns <= 8) rc = up(std::integral_constant<int, 8>());
    else rc = up(std::integral_constant<int, 16>());
    if (rc != CMX_OK) return rc;
    const auto rows = [&](auto rt) -> int {
        const uint32_t down_columns = per_expert(down_most, 2) && a.down_pass > 2 ? 2 : (per_expert(down_most, 4) && a.down_pass > 4 ? 4 : a.down_pass);
        if (down_columns <= 1) return down(rt, std::integral_constant<int, 1>());
        if (down_columns <= 2) return down(rt, std::integral_constant<int, 2>());
        if (down_columns <= 4) return down(rt, std::integral_constant<int, 4>());
        return down(rt, std::integral_constant<int, 8>());
    };
    // Two row tiles share a reading of the activations from LDS, if that leaves workgroups for more than half of the CUs (both matmuls, two tiles and one: 32 tokens,
    // 256 experts, k = 7168 714 us and 774; 12 tokens, 64 experts, k = 5120 195 and 203; 31 tokens, 16 experts, k = 4992 126 and 146; 20 tokens, 128
    // experts, k = 4096 158 and 124).
    return ceil_div(k, 16) > (uint32_t)cus ? rows(std::integral_constant<int, 2>()) : rows(std::integral_constant<int, 1>());
}
