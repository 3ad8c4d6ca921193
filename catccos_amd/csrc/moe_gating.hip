// Routing of tokens to experts: scores of the gate's logits, choice of the best experts, their weights.
//
//   s = softmax(z) or sigmoid(z),   c = s + bias
//   groups: the top_groups groups with the largest sum of their group_best (1 or 2) largest c;  the top_k largest c among their
//   members, ties to the lower index;   weight = s (not c), over its sum if renormalised, times scale
//
// Whole numbers come out, so the order must be that of the exact values, not of their roundings:
//   - without a bias, and with one value for each group, the order of the scores is the order of the logits, which is compared
//     as it is; scores are computed for the chosen experts alone (softmax, not renormalised: the sum over all in addition);
//   - otherwise c is compared in fp32, and values that lie closer than fp32 can tell apart (score_loss), other than by equal logits and biases, are
//     compared again in 64 bits: the groups next to the border between kept and not, the chosen and the first behind them, and the whole row where
//     that may not be all.  With N(0, 1) logits and sigmoids one row in two thousand has such a pair; softmax with a bias has more of them where a few scores
//     are large (8192 rows of 256: 13 us, of 3 x N(0, 1) logits 20).
// Work split: LPR lanes hold a row, so that a wavefront works on 64 / LPR rows at a time; an expert is one key of 64 bits that
// carries value and index.  With 16 lanes to a row the few experts that can be chosen at all are put in a list and count each other; with 64 a round
// of the choice is one maximum over the lanes' own best keys.
// Bound by the vector ALU where there are many rows: 1270 instructions for four rows of 256 in 8 groups, which keep it busy for 78 % of the time.  32768 such
// rows take 27 us (their 17 MB would take 3), 8192 rows of fp32 logits without groups 6.2, one row 5.1, of which a launch is 2.5.
#include <type_traits>

#include "mx_launch.h"

namespace cmx {
namespace {

constexpr uint32_t kWaves = 4, kMaxTopK = 64, kMaxGroups = 64, kMaxExperts = 1024;

// How far an fp32 score as the choice computes it may be off, in units of 2^-24.  Softmax, d = max - z: the difference, the product with log2(e) and that
// constant's own rounding cost 2.3 d of the score, exp2 2, a division and a product 2, the sum that divides 35 additions (32 in a lane, then pairs) and what its
// terms are off, their d on average no more than ln(1024): 18.  (2.3 d + 57) s is below 2^-17 s to d = 30, what it is more from there on below kSumLoss s + kTiny;
// and it is below 2^-18 of the row's largest score for any d.  Sigmoid: exp2, one addition, one reciprocal: s (1 - s) (1.3 |z| + 2) + 3 s, below 2^-22 for any z, and
// (1.3 |z| + 5) s, below 2^-18 of a small s to |z| = 45, what it is more from there on below kTiny.
constexpr float kSumLoss = 0x1p-22f, kTiny = 0x1p-70f;
__device__ __forceinline__ float score_loss(float s, bool softmax) { return softmax ? 0x1p-17f * s : fminf(0x1p-22f, 0x1p-18f * s); }
// of any score of a row
__device__ __forceinline__ float widest_loss(float largest, bool softmax) { return softmax ? 0x1p-18f * largest : 0x1p-22f; }

struct GateArgs {
    const uint8_t* logits;
    size_t ld;                 // bytes
    const float* bias;         // may be null
    int32_t* idx;
    float* weight;
    uint32_t tokens, experts, top_k, groups, members, top_groups, group_best;
    uint32_t by_members;       // ceil(2^20 / members): expert e is in group e * by_members >> 20 (exact: e and members are at most 1024)
    float scale;
    int type, softmax, renormalize;
    int by_logit;              // the order of the logits is the order of the choice
};

__device__ __forceinline__ float logit(const GateArgs& a, const uint8_t* row, uint32_t e) {
    if (a.type == CMX_OUT_FP32) return reinterpret_cast<const float*>(row)[e];
    const uint16_t bits = reinterpret_cast<const uint16_t*>(row)[e];
    return a.type == CMX_OUT_BF16 ? bf16_to_f32(bits) : (float)__builtin_bit_cast(_Float16, bits);
}

// ---- order of floats as whole numbers: 0 is left for experts that cannot be chosen; NaN counts as -Inf
__device__ __forceinline__ uint32_t ord(float f) {
    const uint32_t u = __float_as_uint(fmaxf(f, -INFINITY) + 0.0f);    // (-0 counts as 0)
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unord(uint32_t o) { return __uint_as_float((int)o < 0 ? o & 0x7FFFFFFFu : ~o); }

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
// Butterflies over the 16 or 64 lanes of a row: DPP inside 16 lanes, lane exchanges across them.  op(a, b) gets a lane's value and another's.
template <class Op>
__device__ __forceinline__ uint32_t across(uint32_t v, const Op& op, bool half) {
    const auto r = half ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return op(r[0], r[1]);
}
template <int LPR, class Op>
__device__ __forceinline__ uint32_t butterfly(uint32_t v, const Op& op) {
    v = op(v, dpp<0xB1>(v));                                            // lane ^ 1
    v = op(v, dpp<0x4E>(v));                                            // lane ^ 2
    v = op(v, dpp<0x141>(v));                                           // mirrored in 8
    v = op(v, dpp<0x140>(v));                                           // mirrored in 16
    if constexpr (LPR == 64) {
        v = across(v, op, false);
        v = across(v, op, true);
    }
    return v;
}
template <int LPR>
__device__ __forceinline__ float row_sum(float f) {
    return __uint_as_float(butterfly<LPR>(__float_as_uint(f), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
// the largest value that is a number, -Inf if there is none
template <int LPR>
__device__ __forceinline__ float row_max(float f) {
    return __uint_as_float(butterfly<LPR>(__float_as_uint(f), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    return butterfly<LPR>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    return __hiloint2double((int)dpp<CTRL>((uint32_t)__double2hiint(v)), (int)dpp<CTRL>((uint32_t)__double2loint(v)));
}
template <int LPR>
__device__ __forceinline__ double row_max_key(double v) {
    v = max_key(v, dpp<0xB1>(v));
    v = max_key(v, dpp<0x4E>(v));
    v = max_key(v, dpp<0x141>(v));
    v = max_key(v, dpp<0x140>(v));
    if constexpr (LPR == 64) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t lo = (uint32_t)__double2loint(v), hi = (uint32_t)__double2hiint(v);
            const auto l = half ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false) : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
            const auto h = half ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false) : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
            v = max_key(__hiloint2double((int)h[0], (int)l[0]), __hiloint2double((int)h[1], (int)l[1]));
        }
    }
    return v;
}

__device__ __forceinline__ float sigmoid(float z) {
    const bool small = z < -80.0f;                                      // (exp(-z) may overflow where the score does not)
    const float e = expf(small ? z : -z);
    return small ? e : 1.0f / (1.0f + e);
}
// what the choice makes do with (score_loss)
__device__ __forceinline__ float quick_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ float quick_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + quick_exp(-z)); }

// ---- the choice of one row in 64 bits, by a whole wavefront; `value` holds `experts` doubles of LDS, `group_value` one for each group
__device__ __forceinline__ bool better(double a, uint32_t i, double b, uint32_t j) { return a > b || (a == b && i < j); }
__device__ __forceinline__ double number(double v) { return fmax(v, -INFINITY); }            // NaN counts as -Inf

// c of expert e in 64 bits; softmax: under the row's largest logit and sum of exponentials
__device__ __forceinline__ double exact_choice(const GateArgs& a, const uint8_t* row, uint32_t e, double most, double sum) {
    const double z = logit(a, row, e);
    const double s = !a.softmax ? 1.0 / (1.0 + exp(-z)) : (z == -INFINITY || sum == 0.0 ? 0.0 : exp(z - most) / sum);
    return number(s + (a.bias ? (double)a.bias[e] : 0.0));
}
// most and sum of exact_choice, by a whole wavefront
__device__ __forceinline__ void exact_sum(const GateArgs& a, const uint8_t* row, double& most, double& sum) {
    const uint32_t lane = threadIdx.x & 63;
    most = -INFINITY;
    sum = 0.0;
    if (!a.softmax) return;
    for (uint32_t e = lane; e < a.experts; e += 64) most = fmax(most, (double)logit(a, row, e));
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmax(most, __shfl_xor(most, d));
    for (uint32_t e = lane; e < a.experts; e += 64) {
        const double z = logit(a, row, e);
        if (z != -INFINITY) sum += exp(z - most);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
}
// The groups of `doubtful` that belong to the `wanted` best of them, their values compared in 64 bits, by a whole wavefront; `value`: a double of LDS per group.
__device__ __forceinline__ uint64_t choose_groups_exactly(const GateArgs& a, const uint8_t* row, uint64_t doubtful, uint32_t wanted, double* value) {
    const uint32_t lane = threadIdx.x & 63;
    double most, sum;
    exact_sum(a, row, most, sum);
    for (uint64_t left = doubtful; left; left &= left - 1) {
        const uint32_t g = (uint32_t)__builtin_ctzll(left);
        double first = -INFINITY, second = -INFINITY;
        for (uint32_t j = lane; j < a.members; j += 64) {
            const double v = exact_choice(a, row, g * a.members + j, most, sum);
            second = fmax(second, fmin(first, v));
            first = fmax(first, v);
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double f = __shfl_xor(first, d), s = __shfl_xor(second, d);
            second = fmax(fmax(second, s), fmin(first, f));
            first = fmax(first, f);
        }
        if (lane == 0) value[g] = a.group_best == 2 && a.members > 1 ? number(first + second) : first;
    }
    __builtin_amdgcn_wave_barrier();
    const bool mine = doubtful >> lane & 1ull;
    uint32_t rank = 0;
    for (uint64_t left = doubtful; left; left &= left - 1) {
        const uint32_t h = (uint32_t)__builtin_ctzll(left);
        if (mine && h != lane) rank += better(value[h], h, value[lane], lane);
    }
    return __ballot(mine && rank < wanted);
}

__device__ __forceinline__ void choose_exactly(const GateArgs& a, const uint8_t* row, double* value, double* group_value, uint2* picks) {
    const uint32_t lane = threadIdx.x & 63;
    double most, sum;
    exact_sum(a, row, most, sum);
    for (uint32_t e = lane; e < a.experts; e += 64) value[e] = exact_choice(a, row, e, most, sum);
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
            group_value[lane] = a.group_best == 2 && two ? number(first + second) : first;
        }
        __builtin_amdgcn_wave_barrier();
        uint32_t rank = 0;
        if (lane < a.groups)
            for (uint32_t g = 0; g < a.groups; ++g) rank += g != lane && better(group_value[g], g, group_value[lane], lane);
        kept = __ballot(lane < a.groups && rank < a.top_groups);
    }
    if (!a.bias) {                                                      // the order of the logits, also where 64 bits round their scores to one or to zero
        for (uint32_t e = lane; e < a.experts; e += 64) value[e] = number((double)logit(a, row, e));
        __builtin_amdgcn_wave_barrier();
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

// LDS of a wavefront, in the order in which it lies: doubles first
template <int LPR, int SLOTS>
struct GateLds {
    static constexpr uint32_t kRows = 64 / LPR, kCapacity = LPR * SLOTS, kList = LPR == 16 ? 64 : 0;      // candidates of a row
    static constexpr uint32_t kOrdWords = kRows * kCapacity > 2 * kCapacity ? kRows * kCapacity : 2 * kCapacity;
    uint32_t list, scores, picks, ords, group_values, losses, bytes;
    __host__ __device__ constexpr GateLds(uint32_t groups, uint32_t top_k)
        : list(groups * 8),                                             // group values in 64 bits before it
          scores(list + kRows * kList * 8),
          picks(scores + kRows * (top_k + 2) * 8),
          ords(picks + kRows * (top_k + 2) * 8),
          group_values(ords + kOrdWords * 4),
          losses(group_values + kRows * groups * 4),
          bytes((losses + kRows * groups * 4 + 7) & ~7u) {}
};

// LPR lanes per row, SLOTS experts per lane
template <int LPR, int SLOTS>
__global__ __launch_bounds__(64 * kWaves) void moe_gating_kernel(const GateArgs a) {
    constexpr int kRows = 64 / LPR, kCapacity = LPR * SLOTS, kChunk = SLOTS < 4 ? SLOTS : 4;
    extern __shared__ __attribute__((aligned(8))) uint8_t shared[];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x % LPR, sub = (threadIdx.x & 63) / LPR;
    const uint32_t token = (blockIdx.x * kWaves + wave) * kRows + sub;
    if ((blockIdx.x * kWaves + wave) * kRows >= a.tokens) return;       // (nothing waits for a wavefront)
    const bool live = token < a.tokens;
    const uint8_t* const row = a.logits + (size_t)(live ? token : a.tokens - 1) * a.ld;     // (a row past the last repeats it)
    const GateLds<LPR, SLOTS> lds(a.groups, a.top_k);
    uint8_t* const mine = shared + wave * lds.bytes;
    uint32_t* const ords = reinterpret_cast<uint32_t*>(mine + lds.ords) + sub * kCapacity;              // orders by expert
    const auto picks_of = [&](uint32_t row) { return reinterpret_cast<uint2*>(mine + lds.picks) + row * (a.top_k + 2); };
    uint2* const picks = picks_of(sub);                                                                 // index, order of its value
    float2* const scores = reinterpret_cast<float2*>(mine + lds.scores) + sub * (a.top_k + 2);          // logit, score
    const auto expert = [&](int s) { return (uint32_t)(s / kChunk * kChunk * LPR + lane * kChunk + s % kChunk); };
    const auto bias = [&](uint32_t e) { return a.bias ? a.bias[e] : 0.0f; };
    const auto pick_of = [&](double key) { return make_uint2(min(key_expert(key), a.experts - 1), key_ord(key)); };
    // the bits of a ballot that are this row's
    const auto row_bits = [&](uint64_t all) { return LPR == 64 ? all : all >> (sub * LPR) & ((1ull << (LPR & 63)) - 1); };

    float z[SLOTS], b[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; s += kChunk) {
        const uint32_t e = expert(s);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) b[s + i] = 0.0f;
        if (e + kChunk <= a.experts) {
            if (a.bias) __builtin_memcpy(&b[s], a.bias + e, 4 * kChunk);
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
            for (int i = 0; i < kChunk; ++i) {
                z[s + i] = e + i < a.experts ? logit(a, row, e + i) : -INFINITY;
                if (a.bias && e + i < a.experts) b[s + i] = a.bias[e + i];
            }
        }
    }

    bool poisoned = false;                                              // softmax: a NaN or +Inf makes every score NaN, and the lowest indices are chosen
    float most = -INFINITY, total = 0.0f;
    if (a.softmax) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) poisoned |= !(z[s] < INFINITY);
        poisoned = row_bits(__ballot(poisoned)) != 0;
    }
    if (a.softmax && !(a.by_logit && a.renormalize)) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) most = fmaxf(most, z[s]);
        most = row_max<LPR>(most);
        if (most == -INFINITY) most = 0.0f;                             // (a row of -Inf: scores of zero)
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) total += quick_exp(z[s] - most);
        total = row_sum<LPR>(total);
    }
    // a score that is given away
    const auto score = [&](float v) {
        if (!a.softmax) return sigmoid(v);
        return v == -INFINITY ? 0.0f : expf(v - most) / total;
    };
    uint32_t o[SLOTS];
    const float share = 1.0f / total;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        float c = z[s];
        if (!a.by_logit) {
            c = a.softmax ? (z[s] == -INFINITY ? 0.0f : quick_exp(z[s] - most) * share) : quick_sigmoid(z[s]);
            c = (poisoned ? NAN : c) + b[s];
        }
        o[s] = ord(c);
    }
    if (a.experts < (uint32_t)kCapacity) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) o[s] = expert(s) < a.experts ? o[s] : 0u;
    }

    bool near = false;                                                  // the row is to be done in 64 bits
    uint64_t kept = ~0ull;                                              // groups
    // How far c may be off by its score s.  Two values that are clear of each other have to settle all that lie behind the lower one, so that the allowance must
    // fall along the order of c: without a bias it is the score's own, with one the row's widest.
    const float widest = widest_loss(share, a.softmax);
    const auto choice_loss = [&](float s) { return a.bias ? widest : score_loss(s, a.softmax); };
    if (a.groups > 1) {
        float* const values = reinterpret_cast<float*>(mine + lds.group_values) + sub * a.groups;
        float* const losses = reinterpret_cast<float*>(mine + lds.losses) + sub * a.groups;
        const auto enter = [&](uint32_t g, uint32_t first, uint32_t second) {
            const bool both = a.group_best == 2 && second;
            const float p = unord(first), q = both ? unord(second) : 0.0f;
            values[g] = both ? fmaxf(p + q, -INFINITY) : p;             // (not a NaN)
            losses[g] = 2.0f * choice_loss(p + q) + kSumLoss * (fabsf(p) + fabsf(q));
        };
        const uint32_t over = a.members / kChunk;                       // lanes that a group lies in
        if (kChunk == 4 && a.members % 4 == 0 && (over & (over - 1)) == 0 && over <= (uint32_t)LPR) {
            // the two best of a lane's four, then of 2, 4, ... lanes
#pragma unroll
            for (int s = 0; s < SLOTS; s += kChunk) {
                uint32_t first = 0, second = 0;
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    second = max(second, min(first, o[s + i]));
                    first = max(first, o[s + i]);
                }
                const auto join = [&](uint32_t f, uint32_t g) {
                    second = max(max(second, g), min(first, f));
                    first = max(first, f);
                };
                if (over > 1) join(dpp<0xB1>(first), dpp<0xB1>(second));
                if (over > 2) join(dpp<0x4E>(first), dpp<0x4E>(second));
                if (over > 4) join(dpp<0x141>(first), dpp<0x141>(second));
                if (over > 8) join(dpp<0x140>(first), dpp<0x140>(second));
                if (LPR == 64 && over > 16) join((uint32_t)__shfl_xor((int)first, 16), (uint32_t)__shfl_xor((int)second, 16));
                if (LPR == 64 && over > 32) join((uint32_t)__shfl_xor((int)first, 32), (uint32_t)__shfl_xor((int)second, 32));
                const uint32_t g = expert(s) * a.by_members >> 20;
                if ((lane & (over - 1)) == 0 && g < a.groups) enter(g, first, second);
            }
        } else {                                                        // groups of other sizes: as many lanes for each as there are, a power of two
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) ords[expert(s)] = o[s];
            __builtin_amdgcn_wave_barrier();
            uint32_t team = LPR;
            while (team > 1 && team * a.groups > (uint32_t)LPR) team >>= 1;
            for (uint32_t g0 = 0; g0 < a.groups; g0 += LPR / team) {
                const uint32_t g = g0 + lane / team;
                uint32_t first = 0, second = 0;
                const auto join = [&](uint32_t f, uint32_t g) {
                    second = max(max(second, g), min(first, f));
                    first = max(first, f);
                };
                if (g < a.groups)
                    for (uint32_t j = lane & (team - 1); j < a.members; j += team) join(ords[g * a.members + j], 0);
                if (team > 1) join(dpp<0xB1>(first), dpp<0xB1>(second));
                if (team > 2) join(dpp<0x4E>(first), dpp<0x4E>(second));
                if (team > 4) join(dpp<0x141>(first), dpp<0x141>(second));
                if (team > 8) join(dpp<0x140>(first), dpp<0x140>(second));
                if (LPR == 64 && team > 16) join((uint32_t)__shfl_xor((int)first, 16), (uint32_t)__shfl_xor((int)second, 16));
                if (LPR == 64 && team > 32) join((uint32_t)__shfl_xor((int)first, 32), (uint32_t)__shfl_xor((int)second, 32));
                if ((lane & (team - 1)) == 0 && g < a.groups) enter(g, first, second);
            }
        }
        __builtin_amdgcn_wave_barrier();
        kept = 0;
        float lowest = INFINITY, highest = -INFINITY;                   // of the kept, by the most that they may be too large; of the others, too small
        for (uint32_t g0 = 0; g0 < a.groups; g0 += LPR) {
            const uint32_t g = g0 + lane;
            uint32_t rank = ~0u;
            if (g < a.groups) {
                const float v = values[g];
                rank = 0;
                for (uint32_t h = 0; h < a.groups; ++h) {
                    const float w = values[h];
                    rank += w > v || (w == v && h < g);
                }
                if (rank < a.top_groups) lowest = fminf(lowest, v - losses[g]);
                else highest = fmaxf(highest, v + losses[g]);
            }
            kept |= row_bits(__ballot(rank < a.top_groups)) << g0;
        }
        // groups that fp32 cannot tell from one on the other side of the border: their values in 64 bits decide
        lowest = -row_max<LPR>(-lowest);
        highest = row_max<LPR>(highest);
        near = !a.by_logit && !poisoned && a.top_groups < a.groups && !(lowest > highest + kTiny);
        if (near && a.groups <= (uint32_t)LPR) {
            near = false;
            if (lane < a.groups) near = kept >> lane & 1ull ? !(values[lane] - losses[lane] > highest + kTiny) : !(values[lane] + losses[lane] < lowest - kTiny);
        }
        if (a.groups <= (uint32_t)LPR) {
            uint64_t rows = __ballot(near && live);
            const uint64_t doubtful = rows;
            near = false;
            while (rows) {                                              // every lane of the wavefront sees the same bits
                const uint32_t which = (uint32_t)__builtin_ctzll(rows) / LPR;
                const uint64_t lanes = LPR == 64 ? ~0ull : ((1ull << (LPR & 63)) - 1) << (which * LPR);
                rows &= ~lanes;
                const uint64_t groups = (doubtful & lanes) >> (which * LPR & 63);
                const uint32_t high = __builtin_amdgcn_readlane((uint32_t)(kept >> 32), which * LPR), low = __builtin_amdgcn_readlane((uint32_t)kept, which * LPR);
                const uint64_t sure = ((uint64_t)high << 32 | low) & ~groups;
                const uint32_t t = (blockIdx.x * kWaves + wave) * kRows + which;
                const uint64_t won = choose_groups_exactly(a, a.logits + (size_t)t * a.ld, groups, a.top_groups - (uint32_t)__popcll(sure), reinterpret_cast<double*>(mine));
                if (sub == which) kept = sure | won;
            }
        }
        if (kChunk == 4 && a.members % 4 == 0) {                        // four neighbours are of one group
#pragma unroll
            for (int s = 0; s < SLOTS; s += kChunk) {
                const uint32_t all = kept >> ((expert(s) * a.by_members >> 20) & 63) & 1ull ? ~0u : 0u;
#pragma unroll
                for (int i = 0; i < kChunk; ++i) o[s + i] &= all;
            }
        } else {
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) o[s] = kept >> ((expert(s) * a.by_members >> 20) & 63) & 1ull ? o[s] : 0u;
        }
    }

    // two more than are asked for, to see how near they come
    const uint32_t choices = a.top_groups * a.members, rounds = a.by_logit ? a.top_k : min(a.top_k + 2, choices);
    bool chosen = false;
    if constexpr (LPR == 16) {
        // No more than `rounds` lanes hold larger values than the rounds-th of the lanes' largest, so everything that is chosen is at least that; as a rule
        // little else is.  These candidates go to a list, where each counts the larger ones.
        if (rounds <= 16) {
            constexpr uint32_t kList = GateLds<LPR, SLOTS>::kList;
            double* const list = reinterpret_cast<double*>(mine + lds.list) + sub * kList;
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) top = max(top, o[s]);
            uint32_t larger = 0;
#define CMX_LARGER(I) larger += dpp<0x120 + I>(top) > top;                                    // the lane I places on, around the row
            CMX_LARGER(1) CMX_LARGER(2) CMX_LARGER(3) CMX_LARGER(4) CMX_LARGER(5) CMX_LARGER(6) CMX_LARGER(7) CMX_LARGER(8)
            CMX_LARGER(9) CMX_LARGER(10) CMX_LARGER(11) CMX_LARGER(12) CMX_LARGER(13) CMX_LARGER(14) CMX_LARGER(15)
#undef CMX_LARGER
            const uint32_t least = max(1u, ~row_max<LPR>(larger < rounds ? ~top : 0u));       // the smallest of those with fewer than `rounds` above
            uint32_t count = 0;
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) count += o[s] >= least;
            uint32_t at = count;                                        // of this lane and those before it
            at += dpp<0x111>(at);
            at += dpp<0x112>(at);
            at += dpp<0x114>(at);
            at += dpp<0x118>(at);
            const uint32_t all = row_max<LPR>(at);
            if (__ballot(all > kList || all < rounds) == 0) {
                chosen = true;
                for (uint32_t i = 0; i < kList; i += 16) list[lane + i] = 0.0;
                __builtin_amdgcn_wave_barrier();
                at -= count;
#pragma unroll
                for (int s = 0; s < SLOTS; ++s)
                    if (o[s] >= least) list[at++] = make_key(o[s], expert(s));
                __builtin_amdgcn_wave_barrier();
                const uint32_t longest = max(max(__builtin_amdgcn_readlane(all, 0), __builtin_amdgcn_readlane(all, 16)),
                                             max(__builtin_amdgcn_readlane(all, 32), __builtin_amdgcn_readlane(all, 48)));
                for (uint32_t i0 = 0; i0 < longest; i0 += 32) {
                    const double first = list[i0 + lane], second = list[i0 + 16 + lane];
                    uint32_t place = 0, second_place = 0;
                    for (uint32_t i = 0; i < longest; i += 4) {         // (zeros behind the end)
#pragma unroll
                        for (uint32_t n = 0; n < 4; ++n) {
                            const double k = list[i + n];
                            place += k > first;
                            second_place += k > second;
                        }
                    }
                    if (i0 + lane < all && place < rounds) picks[place] = pick_of(first);
                    if (i0 + 16 + lane < all && second_place < rounds) picks[second_place] = pick_of(second);
                }
            }
        }
    }
    if (!chosen) {
        double key[SLOTS], best = 0.0;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            key[s] = make_key(o[s], expert(s));
            best = max_key(best, key[s]);
        }
        for (uint32_t r = 0; r < rounds; ++r) {
            const double won = row_max_key<LPR>(best);
            if (lane == 0) picks[r] = pick_of(won);
            best = 0.0;
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                key[s] = __double_as_longlong(key[s]) == __double_as_longlong(won) ? 0.0 : key[s];
                best = max_key(best, key[s]);
            }
        }
    }
    __builtin_amdgcn_wave_barrier();

    // logits and scores of the chosen and the one behind them
    if (a.softmax && a.by_logit && a.renormalize) {                     // any common factor is as good as the sum over all
        for (uint32_t r = lane; r < a.top_k; r += LPR) most = fmaxf(most, logit(a, row, picks[r].x));
        most = row_max<LPR>(most);
        total = 1.0f;
    }
    const auto fetch_scores = [&] {
        for (uint32_t r = lane; r < rounds; r += LPR) {
            const float v = logit(a, row, picks[r].x);
            scores[r] = make_float2(v, poisoned ? NAN : score(v));
        }
        __builtin_amdgcn_wave_barrier();
    };
    fetch_scores();
    if (!a.by_logit) {
        // closer than fp32 can tell: values c of scores s
        const auto close = [&](float c, float s, float d, float t) {
            return !(fabsf(c - d) > choice_loss(s) + choice_loss(t) + kSumLoss * (fabsf(c) + fabsf(d)) + kTiny);
        };
        // Neighbours in the order: clear, of equal logits and biases (then the lower index comes first, rightly), or close.  Close ones are put in order
        // by their values in 64 bits, the first that is not chosen among them.  That is all if the second behind is clear of it; if not, more may lie there.
        bool mend = false, border = false, tied = false, open = false;
        for (uint32_t r = lane; r + 1 < rounds; r += LPR) {
            const float2 p = scores[r], q = scores[r + 1];
            const bool same = p.x == q.x && bias(picks[r].x) == bias(picks[r + 1].x);
            const bool unclear = !same && close(unord(picks[r].y), p.y, unord(picks[r + 1].y), q.y);
            mend |= unclear && r < a.top_k;
            border |= (same || unclear) && r + 1 == a.top_k;
            tied |= same && r == a.top_k;
            open |= unclear && r == a.top_k;
        }
        mend = !poisoned && row_bits(__ballot(mend)) != 0;
        border = !poisoned && row_bits(__ballot(border)) != 0;
        tied = border && row_bits(__ballot(tied)) != 0;
        near |= border && row_bits(__ballot(open)) != 0;
        near |= mend && tied;
        if (tied && !mend) {
            const float zl = scores[a.top_k].x, sl = scores[a.top_k].y, bl = bias(picks[a.top_k].x);
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                if (o[s] == 0) continue;
                const float v = logit(a, row, expert(s));
                near |= !(v == zl && bias(expert(s)) == bl) && close(unord(o[s]), score(v), sl + bl, sl);
            }
        }
        const uint64_t rows = __ballot(near && live);
        mend &= row_bits(rows) == 0;
        const uint64_t mended = __ballot(mend);
        if (mended) {
            double sum = 0.0;
            if (a.softmax && a.bias) {
#pragma unroll
                for (int s = 0; s < SLOTS; ++s) sum += expert(s) < a.experts ? exp((double)logit(a, row, expert(s)) - (double)most) : 0.0;
#pragma unroll
                for (int d = 1; d < LPR; d *= 2) sum += __shfl_xor(sum, d);
            }
            const uint32_t entries = mend ? min(a.top_k + 1, rounds) : 0;
            double* const values = reinterpret_cast<double*>(scores);
            uint32_t* const sorted = reinterpret_cast<uint32_t*>(scores);
            for (uint32_t r = lane; r < entries; r += LPR) {            // (each reads the score that it overwrites)
                const double zr = scores[r].x;
                const double v = !a.bias ? zr : (!a.softmax ? 1.0 / (1.0 + exp(-zr)) : zr == -INFINITY ? 0.0 : exp(zr - (double)most) / sum);      // (without a bias the order of the logits)
                values[r] = number(v + (double)bias(picks[r].x));
            }
            __builtin_amdgcn_wave_barrier();
            for (uint32_t r = lane; r < entries; r += LPR) {
                const double v = values[r];
                const uint32_t e = picks[r].x;
                uint32_t place = 0;
                for (uint32_t q = 0; q < entries; ++q) place += q != r && better(values[q], picks[q].x, v, e);
                picks[r].y = place;
            }
            __builtin_amdgcn_wave_barrier();
            for (uint32_t r = lane; r < entries; r += LPR) sorted[picks[r].y] = picks[r].x;
            __builtin_amdgcn_wave_barrier();
            for (uint32_t r = lane; r < entries; r += LPR) picks[r].x = sorted[r];
            __builtin_amdgcn_wave_barrier();
        }
        for (uint64_t left = rows; left;) {                             // every lane of the wavefront sees the same bits
            const uint32_t which = (uint32_t)__builtin_ctzll(left) / LPR;
            left &= LPR == 64 ? 0ull : ~(((1ull << (LPR & 63)) - 1) << (which * LPR));
            const uint32_t t = (blockIdx.x * kWaves + wave) * kRows + which;
            choose_exactly(a, a.logits + (size_t)t * a.ld, reinterpret_cast<double*>(mine + lds.ords), reinterpret_cast<double*>(mine), picks_of(which));
        }
        if (rows | mended) fetch_scores();
    }

    float sum = 0.0f;
    if (a.renormalize) {
        for (uint32_t r = lane; r < a.top_k; r += LPR) sum += scores[r].y;
        sum = row_sum<LPR>(sum);
        // Scores that fp32 holds in part or not at all: their quotients are those of exp(z), under the largest chosen logit.  (Below 2^-23 the 1 of a sigmoid's
        // denominator is all of it.  What 64 bits do not hold either, below exp(-745), stays zero.)
        const bool faint = sum < 0x1p-23f;
        if (__builtin_expect(__ballot(faint) != 0, 0)) {
            float high = -INFINITY;
            for (uint32_t r = lane; r < a.top_k; r += LPR) high = fmaxf(high, scores[r].x);
            high = row_max<LPR>(high);
            if (faint && high - (a.softmax ? most : 0.0f) > -745.0f)
                for (uint32_t r = lane; r < a.top_k; r += LPR) scores[r].y = expf(scores[r].x - high);
            float again = 0.0f;
            for (uint32_t r = lane; r < a.top_k; r += LPR) again += scores[r].y;
            sum = row_sum<LPR>(again);
        }
    }
    for (uint32_t r = lane; r < a.top_k && live; r += LPR) {
        const float s = scores[r].y;
        a.idx[(size_t)token * a.top_k + r] = (int32_t)picks[r].x;
        a.weight[(size_t)token * a.top_k + r] = (!a.renormalize ? s : sum == 0.0f ? 0.0f : s / sum) * a.scale;
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
    CMX_REQUIRE((uint64_t)tokens * top_k < (1ull << 31) && fits_grid((uint64_t)tokens + 3, 64), "tokens must stay below 2^26, tokens * top_k below 2^31 routes");
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
                        experts / groups, top_groups, group_best, ceil_div(1u << 20, experts / groups), scale, type, score == CMX_SCORE_SOFTMAX, renormalize != 0,
                        !bias && (groups == 1 || group_best == 1 || experts == groups)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const auto run = [&](auto lanes, auto slots) -> int {
        const GateLds<lanes.value, slots.value> lds(groups, top_k);
        constexpr size_t kMostLds = kWaves * GateLds<lanes.value, slots.value>(kMaxGroups, kMaxTopK).bytes;
        if constexpr (kMostLds > 64 * 1024) {                           // (512 experts, 64 groups and top_k 64 by 16 lanes: 66.5 KiB)
            if (int rc = allow_dynamic_lds<moe_gating_kernel<lanes.value, slots.value>, kMostLds>(); rc != CMX_OK) return rc;
        }
        hipLaunchKernelGGL((moe_gating_kernel<lanes.value, slots.value>), dim3(ceil_div(tokens, 64 / lanes.value * kWaves)), dim3(64 * kWaves),
                           kWaves * lds.bytes, s, a);
        CMX_LAUNCH_CHECK();
        return CMX_OK;
    };
    using std::integral_constant;
    const auto by_slots = [&](auto lanes) -> int {
        const uint32_t slots = ceil_div(experts, lanes.value);
        if (slots <= 1) return run(lanes, integral_constant<int, 1>());
        if (slots <= 2) return run(lanes, integral_constant<int, 2>());
        if (slots <= 4) return run(lanes, integral_constant<int, 4>());
        if (slots <= 8) return run(lanes, integral_constant<int, 8>());
        if (slots <= 16 || lanes.value == 64) return run(lanes, integral_constant<int, 16>());
        return run(lanes, integral_constant<int, lanes.value == 16 ? 32 : 16>());
    };
    // 16 lanes to a row do less work, 64 are done sooner.  Measured in a graph, 64 and 16 lanes, softmax top-8 of 256 / sigmoid in 8 groups: 1024 rows 5.3 and
    // 6.0 / 7.0 and 9.9 us, 4096 rows 7.1 and 6.2 / 10.9 and 10.0, on 256 CUs; of 512, 4096 rows 10.5 and 10.0 / 14.9 and 15.3, 32768
    // rows 43.6 and 28.4 / 63.5 and 43.1.
    int cus;
    if (int rc = cu_count(&cus); rc != CMX_OK) return rc;
    if (tokens >= 14u * (uint32_t)cus && experts <= 512) return by_slots(integral_constant<int, 16>());
    return by_slots(integral_constant<int, 64>());
}
