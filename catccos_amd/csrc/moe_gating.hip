// Routing of tokens to experts: scores of the gate's logits, choice of the best experts, their weights.
//
//   s = softmax(z) or sigmoid(z),   c = s + bias
//   groups: the top_groups groups with the largest sum of their group_best (1 or 2) largest c;  the top_k largest c among their
//   members, ties to the lower index;   weight = s (not c), over its sum if renormalised, times scale
//
// Whole numbers come out, so the order must be that of the exact values, not of their roundings:
//   - without a bias, and with one value for each group, the order of the scores is the order of the logits, which is compared
//     as it is; scores are computed for the chosen experts alone (softmax, not renormalised: the sum over all in addition);
//   - otherwise c is compared in fp32, and a row in which two values lie closer than fp32 can tell apart (kSoftmaxLoss, kSigmoidLoss), other
//     than by equal logits and biases, is done again in 64 bits by its whole wavefront.
// Work split: LPR lanes hold a row, so that a wavefront works on 64 / LPR rows at a time; an expert is one key of 64 bits that
// carries value and index, and a round of the choice is one maximum over the lanes' own best keys.
#include "mx_common.h"

namespace cmx {
namespace {

constexpr uint32_t kWaves = 4, kMaxTopK = 64, kMaxGroups = 64, kMaxExperts = 1024;

// Relative error of an fp32 score.  Softmax: exp of z - max (its rounding alone costs |z - max| * 2^-24, and 64 * 2^-24 is reached where the score
// is 10^-28), sums of up to 1024 terms (16 in a lane, then pairs), one division: below 2^-17.  Sigmoid: exp, one addition, one division: below 2^-21.
constexpr float kSoftmaxLoss = 0x1p-17f, kSigmoidLoss = 0x1p-21f, kSumLoss = 0x1p-22f, kTiny = 0x1p-90f;

struct GateArgs {
    const uint8_t* logits;
    size_t ld;                 // bytes
    const float* bias;         // may be null
    int32_t* idx;
    float* weight;
    uint32_t tokens, experts, top_k, groups, members, top_groups, group_best;
    float scale;
    int type, softmax, renormalize;
    int by_logit;              // the order of the logits is the order of the choice
};

__device__ __forceinline__ float logit(const GateArgs& a, const uint8_t* row, uint32_t e) {
    if (a.type == CMX_OUT_FP32) return reinterpret_cast<const float*>(row)[e];
    const uint16_t bits = reinterpret_cast<const uint16_t*>(row)[e];
    return a.type == CMX_OUT_BF16 ? bf16_to_f32(bits) : (float)__builtin_bit_cast(_Float16, bits);
}

// ---- order of floats as whole numbers: 0 is left for experts that cannot be chosen, 1 is any NaN, -Inf and upwards lie above
__device__ __forceinline__ uint32_t ord(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);                      // (-0 counts as 0)
    return f != f ? 1u : ((int)u < 0 ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ float unord(uint32_t o) {
    return o <= 1u ? __uint_as_float(0x7FC00000u) : __uint_as_float((int)o < 0 ? o & 0x7FFFFFFFu : ~o);
}

// ---- keys: order above, index below (the lower index is the larger key), in the mantissa of a double from [1, 2), whose maximum is one instruction
__device__ __forceinline__ double make_key(uint32_t o, uint32_t e) {
    return __hiloint2double((int)(0x3FF00000u | (o >> 22)), (int)((o << 10) | (kMaxExperts - 1 - e)));
}
__device__ __forceinline__ uint32_t key_expert(double k) { return kMaxExperts - 1 - ((uint32_t)__double2loint(k) & (kMaxExperts - 1)); }
__device__ __forceinline__ uint32_t key_ord(double k) { return ((uint32_t)__double2hiint(k) << 22) | ((uint32_t)__double2loint(k) >> 10); }
__device__ __forceinline__ double max_key(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));             // (never a NaN: no canonicalisation in front)
    return r;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
// the lanes' other value under one step of a butterfly over 64 lanes: step 0..3 inside rows of 16, 4 and 5 across them
template <int STEP>
__device__ __forceinline__ uint32_t partner(uint32_t v) {
    if constexpr (STEP == 0) return dpp<0xB1>(v);                       // lane ^ 1
    if constexpr (STEP == 1) return dpp<0x4E>(v);                       // lane ^ 2
    if constexpr (STEP == 2) return dpp<0x141>(v);                      // mirrored in 8
    if constexpr (STEP == 3) return dpp<0x140>(v);                      // mirrored in 16
    return (uint32_t)__shfl_xor((int)v, STEP == 4 ? 16 : 32);
}
template <int STEP>
__device__ __forceinline__ double partner(double v) {
    return __hiloint2double((int)partner<STEP>((uint32_t)__double2hiint(v)), (int)partner<STEP>((uint32_t)__double2loint(v)));
}
template <int LPR>
__device__ __forceinline__ double row_max_key(double v) {
    v = max_key(v, partner<0>(v));
    v = max_key(v, partner<1>(v));
    v = max_key(v, partner<2>(v));
    v = max_key(v, partner<3>(v));
    if constexpr (LPR == 64) {
        v = max_key(v, partner<4>(v));
        v = max_key(v, partner<5>(v));
    }
    return v;
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
    v += __uint_as_float(partner<0>(__float_as_uint(v)));
    v += __uint_as_float(partner<1>(__float_as_uint(v)));
    v += __uint_as_float(partner<2>(__float_as_uint(v)));
    v += __uint_as_float(partner<3>(__float_as_uint(v)));
    if constexpr (LPR == 64) {
        v += __uint_as_float(partner<4>(__float_as_uint(v)));
        v += __uint_as_float(partner<5>(__float_as_uint(v)));
    }
    return v;
}
// the largest value that is a number, -Inf if there is none
template <int LPR>
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, __uint_as_float(partner<0>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(partner<1>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(partner<2>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(partner<3>(__float_as_uint(v))));
    if constexpr (LPR == 64) {
        v = fmaxf(v, __uint_as_float(partner<4>(__float_as_uint(v))));
        v = fmaxf(v, __uint_as_float(partner<5>(__float_as_uint(v))));
    }
    return v;
}

__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }

// ---- the choice of one row in 64 bits, by a whole wavefront; `value` holds `experts` doubles of LDS, `group_value` one for each group
__device__ __forceinline__ bool better(double a, uint32_t i, double b, uint32_t j) {          // NaN behind everything
    if (a != a || b != b) return a != a ? (b != b && i < j) : true;
    return a > b || (a == b && i < j);
}

__device__ __forceinline__ void choose_exactly(const GateArgs& a, const uint8_t* row, double* value, double* group_value, uint2* picks) {
    const uint32_t lane = threadIdx.x & 63;
    double most = -INFINITY, sum = 0.0;
    if (a.softmax) {
        for (uint32_t e = lane; e < a.experts; e += 64) most = fmax(most, (double)logit(a, row, e));
        for (int d = 32; d > 0; d >>= 1) most = fmax(most, __shfl_xor(most, d));
        for (uint32_t e = lane; e < a.experts; e += 64) {
            const double z = logit(a, row, e);
            const double v = z == -INFINITY ? 0.0 : exp(z - most);
            value[e] = v;
            sum += v;
        }
        for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    }
    for (uint32_t e = lane; e < a.experts; e += 64) {
        const double s = a.softmax ? (sum == 0.0 ? 0.0 : value[e] / sum) : 1.0 / (1.0 + exp(-(double)logit(a, row, e)));
        value[e] = s + (a.bias ? (double)a.bias[e] : 0.0);
    }
    __builtin_amdgcn_wave_barrier();
    uint64_t kept = ~0ull;
    if (a.groups > 1) {
        double first = -INFINITY, second = -INFINITY;
        bool any = false, two = false;
        if (lane < a.groups) {
            for (uint32_t j = 0; j < a.members; ++j) {
                const double v = value[lane * a.members + j];
                if (!any || better(v, 0, first, 1)) {
                    second = first;
                    two = any;
                    first = v;
                    any = true;
                } else if (!two || better(v, 0, second, 1)) {
                    second = v;
                    two = true;
                }
            }
            group_value[lane] = a.group_best == 2 && two ? first + second : first;
        }
        __builtin_amdgcn_wave_barrier();
        uint32_t rank = 0;
        if (lane < a.groups)
            for (uint32_t g = 0; g < a.groups; ++g) rank += g != lane && better(group_value[g], g, group_value[lane], lane);
        kept = __ballot(lane < a.groups && rank < a.top_groups);
    }
    uint32_t taken = 0;                                                 // of this lane's experts lane, lane + 64, ...
    for (uint32_t r = 0; r < a.top_k; ++r) {
        double best = 0.0;
        uint32_t at = ~0u;
        for (uint32_t e = lane, n = 0; e < a.experts; e += 64, ++n) {
            if ((taken >> n & 1u) || !(kept >> (e / a.members) & 1ull)) continue;
            if (at == ~0u || better(value[e], e, best, at)) {
                best = value[e];
                at = e;
            }
        }
        for (int d = 32; d > 0; d >>= 1) {
            const double v = __shfl_xor(best, d);
            const uint32_t e = (uint32_t)__shfl_xor((int)at, d);
            if (e != ~0u && (at == ~0u || better(v, e, best, at))) {
                best = v;
                at = e;
            }
        }
        if ((at & 63) == lane) taken |= 1u << (at >> 6);
        if (lane == 0) picks[r] = make_uint2(at, 0);
    }
    __builtin_amdgcn_wave_barrier();
}

// LPR lanes per row, SLOTS experts per lane
template <int LPR, int SLOTS>
__global__ __launch_bounds__(64 * kWaves) void moe_gating_kernel(const GateArgs a) {
    constexpr int kRows = 64 / LPR, kCapacity = LPR * SLOTS, kChunk = SLOTS < 4 ? SLOTS : 4;
    constexpr int kOrdWords = kRows * kCapacity > 2 * kCapacity ? kRows * kCapacity : 2 * kCapacity;
    __shared__ __attribute__((aligned(8))) uint32_t ords_[kWaves][kOrdWords];
    __shared__ double group_values_[kWaves][kMaxGroups];
    __shared__ uint32_t group_ords_[kWaves][kRows][kMaxGroups];
    __shared__ uint2 picks_[kWaves][kRows][kMaxTopK + 1];               // index, order of its value
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x % LPR, sub = (threadIdx.x & 63) / LPR;
    const uint32_t token = (blockIdx.x * kWaves + wave) * kRows + sub;
    if ((blockIdx.x * kWaves + wave) * kRows >= a.tokens) return;       // (nothing waits for a wavefront)
    const bool live = token < a.tokens;
    const uint8_t* const row = a.logits + (size_t)(live ? token : a.tokens - 1) * a.ld;     // (a row past the last repeats it)
    uint32_t* const ords = ords_[wave] + sub * kCapacity;
    uint2* const picks = picks_[wave][sub];
    const auto expert = [&](int s) { return (uint32_t)(s / kChunk * kChunk * LPR + lane * kChunk + s % kChunk); };

    float z[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; s += kChunk) {
        const uint32_t e = expert(s);
        if (e + kChunk <= a.experts) {
            if (a.type == CMX_OUT_FP32) {
                __builtin_memcpy(&z[s], row + (size_t)e * 4, 4 * kChunk);
            } else {
                uint16_t h[kChunk];
                __builtin_memcpy(h, row + (size_t)e * 2, 2 * kChunk);
#pragma unroll
                for (int i = 0; i < kChunk; ++i) z[s + i] = a.type == CMX_OUT_BF16 ? bf16_to_f32(h[i]) : (float)__builtin_bit_cast(_Float16, h[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) z[s + i] = e + i < a.experts ? logit(a, row, e + i) : -INFINITY;
        }
    }

    bool poisoned = false;                                              // softmax: a NaN or +Inf makes every score NaN
    float most = -INFINITY, total = 0.0f;
    if (a.softmax) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) poisoned |= !(z[s] < INFINITY);
        poisoned = (__ballot(poisoned) >> (sub * LPR) & (LPR == 64 ? ~0ull : (1ull << (LPR & 63)) - 1)) != 0;
    }
    if (a.softmax && !(a.by_logit && a.renormalize)) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) most = fmaxf(most, z[s]);
        most = row_max<LPR>(most);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) total += z[s] == -INFINITY ? 0.0f : expf(z[s] - most);
        total = row_sum<LPR>(total);
    }
    // a score of fp32
    const auto score = [&](float v) {
        if (!a.softmax) return sigmoid(v);
        return v == -INFINITY ? 0.0f : expf(v - most) / total;
    };
    uint32_t o[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const uint32_t e = expert(s);
        float c = z[s];
        if (!a.by_logit) c = (poisoned ? NAN : score(z[s])) + (a.bias && e < a.experts ? a.bias[e] : 0.0f);
        o[s] = e < a.experts ? ord(c) : 0u;
    }

    bool near = false;                                                  // two values that fp32 cannot tell apart
    if (a.groups > 1) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) ords[expert(s)] = o[s];
        __builtin_amdgcn_wave_barrier();
        uint32_t* const group_ords = group_ords_[wave][sub];
        for (uint32_t g = lane; g < a.groups; g += LPR) {
            uint32_t first = 0, second = 0, j = g % a.members;          // (each lane starts elsewhere: no two read one bank)
            for (uint32_t n = 0; n < a.members; ++n) {
                const uint32_t v = ords[g * a.members + j];
                j = j + 1 == a.members ? 0 : j + 1;
                second = max(second, min(first, v));
                first = max(first, v);
            }
            group_ords[g] = a.group_best == 2 && second ? ord(unord(first) + unord(second)) : first;
        }
        __builtin_amdgcn_wave_barrier();
        // how far a sum of two scores (each at most 1) and their biases may be off
        const float loss = 2.0f * (a.softmax ? kSoftmaxLoss : kSigmoidLoss);
        for (uint32_t g = lane; g < a.groups; g += LPR) {
            const uint32_t mine = group_ords[g];
            const float v = unord(mine);
            uint32_t rank = 0;
            for (uint32_t h = 0; h < a.groups; ++h) {
                const uint32_t other = group_ords[h];
                const float w = unord(other);
                rank += other > mine || (other == mine && h < g);
                near |= !a.by_logit && h != g && !(fabsf(v - w) > 2.0f * loss + 4.0f * kSumLoss * (fabsf(v) + fabsf(w) + 1.0f));
            }
            if (rank >= a.top_groups)
                for (uint32_t j = 0; j < a.members; ++j) ords[g * a.members + j] = 0;
        }
        near &= a.top_groups < a.groups;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) o[s] = ords[expert(s)];
    }

    double key[SLOTS], best = 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        key[s] = make_key(o[s], expert(s));
        best = max_key(best, key[s]);
    }
    // one more than is asked for, to see how near it comes
    const uint32_t choices = a.top_groups * a.members, rounds = a.by_logit ? a.top_k : min(a.top_k + 1, choices);
    for (uint32_t r = 0; r < rounds; ++r) {
        const double won = row_max_key<LPR>(best);
        if (lane == 0) picks[r] = make_uint2(key_expert(won), key_ord(won));
        best = 0.0;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            key[s] = __double_as_longlong(key[s]) == __double_as_longlong(won) ? 0.0 : key[s];
            best = max_key(best, key[s]);
        }
    }
    __builtin_amdgcn_wave_barrier();
    if (!a.by_logit) {
        // closer than fp32 can tell: values c of scores s
        const float loss = a.softmax ? kSoftmaxLoss : kSigmoidLoss;
        const auto close = [&](float c, float s, float d, float t) { return !(fabsf(c - d) > loss * (s + t) + kSumLoss * (fabsf(c) + fabsf(d)) + kTiny); };
        const auto bias = [&](uint32_t e) { return a.bias ? a.bias[e] : 0.0f; };
        // Neighbours in the order: of equal logits and biases the lower index comes first, rightly.  Where the last chosen and the first that is
        // not are such a pair, any other value beside them may lie further down, so all are looked at.
        bool tied = false;
        for (uint32_t r = lane; r + 1 < rounds; r += LPR) {
            const uint2 p = picks[r], q = picks[r + 1];
            const float zp = logit(a, row, p.x), zq = logit(a, row, q.x);
            const bool same = zp == zq && bias(p.x) == bias(q.x);
            near |= !same && close(unord(p.y), score(zp), unord(q.y), score(zq));
            tied |= same && r + 1 == a.top_k;
        }
        tied = (__ballot(tied) >> (sub * LPR) & (LPR == 64 ? ~0ull : (1ull << (LPR & 63)) - 1)) != 0;
        if (tied) {
            const uint32_t last = picks[a.top_k].x;
            const float zl = logit(a, row, last), sl = score(zl), bl = bias(last);
            for (uint32_t e = lane; e < a.experts; e += LPR) {
                if (a.groups > 1 && ords[e] == 0) continue;
                const float z = logit(a, row, e), s = score(z), b = bias(e);
                near |= !(z == zl && b == bl) && close(s + b, s, sl + bl, sl);
            }
        }
        uint64_t rows = __ballot(near && live);
        while (rows) {                                                  // every lane of the wavefront sees the same bits
            const uint32_t which = (uint32_t)__builtin_ctzll(rows) / LPR;
            rows &= LPR == 64 ? 0ull : ~(((1ull << (LPR & 63)) - 1) << (which * LPR));
            const uint32_t t = (blockIdx.x * kWaves + wave) * kRows + which;
            choose_exactly(a, a.logits + (size_t)t * a.ld, reinterpret_cast<double*>(ords_[wave]), group_values_[wave], picks_[wave][which]);
        }
        __builtin_amdgcn_wave_barrier();
    }

    // weights: scores of the chosen
    if (a.softmax && a.by_logit && a.renormalize) {                     // any common factor is as good as the sum over all
        for (uint32_t r = lane; r < a.top_k; r += LPR) most = fmaxf(most, logit(a, row, picks[r].x));
        most = row_max<LPR>(most);
        total = 1.0f;
    }
    float mine[kMaxTopK / LPR], sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kMaxTopK / LPR; ++i) {
        const uint32_t r = lane + i * LPR;
        mine[i] = 0.0f;
        if (r < a.top_k) mine[i] = poisoned ? NAN : score(logit(a, row, picks[r].x));
        sum += mine[i];
    }
    if (a.renormalize) sum = row_sum<LPR>(sum);
#pragma unroll
    for (uint32_t i = 0; i < kMaxTopK / LPR; ++i) {
        const uint32_t r = lane + i * LPR;
        if (r >= a.top_k || !live) continue;
        a.idx[(size_t)token * a.top_k + r] = (int32_t)picks[r].x;
        a.weight[(size_t)token * a.top_k + r] = (!a.renormalize ? mine[i] : sum == 0.0f ? 0.0f : mine[i] / sum) * a.scale;
    }
}

}  // namespace
}  // namespace cmx

int cmx::preload_gating_kernels() {
    hipFuncAttributes attr;
    CMX_HIP(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(cmx::moe_gating_kernel<64, 1>)));
    return CMX_OK;
}

extern "C" int cmx_moe_gating(const void* logits, uint32_t ld_logits, int type, const float* bias, uint32_t tokens, uint32_t experts,
                              uint32_t top_k, int score, uint32_t groups, uint32_t top_groups, uint32_t group_best, int renormalize,
                              uint32_t scale_bits, int32_t* expert_idx, float* gate_weight, cmx_stream_t stream) {
    using namespace cmx;
    CMX_REQUIRE(type == CMX_OUT_BF16 || type == CMX_OUT_FP16 || type == CMX_OUT_FP32, "unknown type");
    CMX_REQUIRE(score == CMX_SCORE_SOFTMAX || score == CMX_SCORE_SIGMOID, "unknown score");
    CMX_REQUIRE(experts > 0 && experts <= kMaxExperts, "experts must be in [1, 1024]");
    CMX_REQUIRE(groups > 0 && groups <= kMaxGroups && experts % groups == 0, "experts must fall into at most 64 groups of one size");
    CMX_REQUIRE(top_groups > 0 && top_groups <= groups, "top_groups must be in [1, groups]");
    CMX_REQUIRE(group_best == 1 || group_best == 2, "group_best must be 1 or 2");
    CMX_REQUIRE(top_k > 0 && top_k <= kMaxTopK && top_k <= top_groups * (experts / groups), "top_k must not exceed 64 or the experts of the chosen groups");
    CMX_REQUIRE((uint64_t)tokens * top_k < (1ull << 31), "tokens * top_k must stay below 2^31 routes");
    float scale;
    __builtin_memcpy(&scale, &scale_bits, 4);
    CMX_REQUIRE(scale - scale == 0.0f, "scale must be a finite number");
    if (tokens == 0) return CMX_OK;
    CMX_REQUIRE(logits && expert_idx && gate_weight, "null pointer");
    CMX_REQUIRE(ld_logits >= experts, "row pitch smaller than row");
    const uint32_t bytes = type == CMX_OUT_FP32 ? 4 : 2;
    CMX_REQUIRE(reinterpret_cast<uintptr_t>(logits) % bytes == 0 && reinterpret_cast<uintptr_t>(bias) % 4 == 0 &&
                reinterpret_cast<uintptr_t>(expert_idx) % 4 == 0 && reinterpret_cast<uintptr_t>(gate_weight) % 4 == 0, "pointers must be aligned to their elements");
    const GateArgs a = {static_cast<const uint8_t*>(logits), (size_t)ld_logits * bytes, bias, expert_idx, gate_weight, tokens, experts, top_k, groups,
                        experts / groups, top_groups, group_best, scale, type, score == CMX_SCORE_SOFTMAX, renormalize != 0,
                        !bias && (groups == 1 || group_best == 1 || experts == groups)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const auto run = [&](auto kernel, uint32_t rows) {
        hipLaunchKernelGGL(kernel, dim3(ceil_div(tokens, rows * kWaves)), dim3(64 * kWaves), 0, s, a);
    };
    if (tokens >= 2048 && experts <= 256) {
        if (experts <= 16) run(moe_gating_kernel<16, 1>, 4);
        else if (experts <= 32) run(moe_gating_kernel<16, 2>, 4);
        else if (experts <= 64) run(moe_gating_kernel<16, 4>, 4);
        else if (experts <= 128) run(moe_gating_kernel<16, 8>, 4);
        else run(moe_gating_kernel<16, 16>, 4);
    } else if (experts <= 64) run(moe_gating_kernel<64, 1>, 1);
    else if (experts <= 128) run(moe_gating_kernel<64, 2>, 1);
    else if (experts <= 256) run(moe_gating_kernel<64, 4>, 1);
    else if (experts <= 512) run(moe_gating_kernel<64, 8>, 1);
    else run(moe_gating_kernel<64, 16>, 1);
    CMX_LAUNCH_CHECK();
    return CMX_OK;
}
