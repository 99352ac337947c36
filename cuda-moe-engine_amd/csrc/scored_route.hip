// Routing by scores: softmax or sigmoid of the logits, a bias that only takes part in the
// choice, groups of experts, top-k, renormalised and scaled weights; and its gradient.
//
//   s = sigmoid(l) or softmax(l);  key = s + bias, or without a bias the logit itself
//   (the same order);  a group's score: the sum of its best one or two s + bias;
//   the best groups, the best keys in them, ties to the lowest index;
//   w = scale s_j / sum_chosen s  or  scale s_j.
//
// A token is a segment of LANES lanes of a wave, V experts a lane, every group in lanes of
// its own. A lane sorts its keys once; each choice is then a maximum over the segment of the lanes' first
// keys, which the owner removes. The choice is by exact value, so that the ids are the definition's and do not
// depend on how exp rounds: keys are fp32 first, and where the order hangs on a difference within their
// rounding, or on a tie, the few experts or the groups that it concerns are compared in 64 bits. That is about one
// token in a thousand at 256 experts; choosing such a token in 64 bits as a whole made 16384 tokens 19 us instead of
// 14, since the wave that does it waits for code that is in no cache. Chosen as a whole are tokens without K
// experts, with infinite keys, NaN, or more than kCandidates like keys, and near ties where a token has
// fewer lanes than that.
//
// Bound by instructions, not bytes: 16384 tokens of 256 experts, top-8 in 4 of 8 groups, are 17.6 MB (3.5 us)
// and 13.8 us; one token 4.2.
#include "row_ops.h"

namespace moe {

namespace {

__device__ __forceinline__ double lane_xor(double x, int mask) { return __shfl_xor(x, mask); }
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }

// The largest over aligned segments of `lanes` lanes, in each lane.
template <int LANES>
__device__ __forceinline__ double segment_max(double x) {
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) x = most(x, lane_xor(x, d));
    return x;
}

// Where a lane's V experts lie.
struct Place {
    int first;   // the lane's first expert
    int count;   // its experts (0: none)
    int lane;    // lane of the token's segment
    int group;   // its group, past the last one without experts
    int group_lanes;  // a power of two
};

// Chooses the token's experts in 64 bits, ties to the lower index: rank[i] = the slot
// of the lane's expert i or -1.
template <int LANES, int V>
__device__ __forceinline__ void choose(const ScoreArgs& a, const Place& p, const float (&l)[V], const float (&b)[V],
                                       int (&rank)[V]) {
    const bool has_bias = a.bias != nullptr;
    double key[V], score[V];
    if (has_bias || a.groups > 1) {
        if (a.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; ++i) score[i] = 1.0 / (1.0 + exp(-static_cast<double>(l[i])));
        } else {
            double top = -__builtin_inf();
#pragma unroll
            for (int i = 0; i < V; ++i) top = most(top, static_cast<double>(l[i]));
            top = segment_max<LANES>(top);
            double total = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                // NaN is out as -inf is and has no part in the others' scores. Logits of +inf (each equal to `top`, where a
                // difference would be NaN) share the whole sum.
                const double x = static_cast<double>(l[i]);
                score[i] = !(l[i] > -__builtin_inff()) ? 0.0 : x == top ? 1.0 : exp(x - top);
                total += score[i];
            }
#pragma unroll
            for (int d = 1; d < LANES; d <<= 1) total += lane_xor(total, d);
#pragma unroll
            for (int i = 0; i < V; ++i) score[i] /= total;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            score[i] += static_cast<double>(b[i]);
            // An expert that is out (a logit of -inf, or no number) has no key.
            if (!(l[i] > -__builtin_inff()) || !(score[i] == score[i])) score[i] = -__builtin_inf();
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        key[i] = has_bias ? score[i] : (l[i] > -__builtin_inff() ? static_cast<double>(l[i]) : -__builtin_inf());
    bool open = true;
    if (a.groups > 1) {
        // The lane's best two, then the group's.
        double first = -__builtin_inf(), second = -__builtin_inf();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < p.count) {
                second = most(second, score[i] < first ? score[i] : first);
                first = most(first, score[i]);
            }
        for (int d = 1; d < p.group_lanes; d <<= 1) {
            const double f = lane_xor(first, d), s = lane_xor(second, d);
            second = most(most(second, s), f < first ? f : first);
            first = most(first, f);
        }
        double group = first;
        if (a.group_best == 2 && second > -__builtin_inf()) group += second;
        // Its place among the groups, ties to the lower one; lanes without a group are last.
        const int mine = p.group;
        const bool real = mine < a.groups;
        int before = 0;
        for (int o = 1; o << a.lane_shift < LANES; ++o) {
            const double other = lane_xor(group, o << a.lane_shift);
            const int index = mine ^ o;
            if (index < a.groups && (other > group || (other == group && index < mine))) ++before;
        }
        open = real && before < a.top_groups;
    }
    // Keys as unsigned integers of the same order. Chosen experts and those of other groups hold 0, as do those
    // that are out, which are chosen last, in order.
    uint64_t order[V];
    uint32_t left = 0;  // experts of the lane that can be chosen
#pragma unroll
    for (int i = 0; i < V; ++i) {
        rank[i] = -1;
        const bool can = open && i < p.count;
        if (can) left |= 1u << i;
        const uint64_t u = __double_as_longlong(key[i] + 0.0);  // -0 is 0
        order[i] = can && key[i] > -__builtin_inf() ? u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | (1ull << 63)) : 0;
    }
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t segment = (LANES == 64 ? ~0ull : ((1ull << (LANES & 63)) - 1)) << (lane / LANES * LANES);
    for (int k = 0; k < a.topk; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) best = order[i] > best ? order[i] : best;
        const uint32_t high = static_cast<uint32_t>(best >> 32);
        const uint32_t top_high = lanes_max<LANES>(high);
        const uint32_t top_low = lanes_max<LANES>(high == top_high ? static_cast<uint32_t>(best) : 0u);
        const uint64_t top = static_cast<uint64_t>(top_high) << 32 | top_low;
        const uint64_t with = __ballot(left != 0 && best == top) & segment;
        if (with >> lane & 1 && (with & ((1ull << lane) - 1)) == 0) {
            bool done = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool take = !done && (left >> i & 1) && order[i] == top;
                rank[i] = take ? k : rank[i];
                order[i] = take ? 0 : order[i];
                left &= take ? ~(1u << i) : ~0u;
                done |= take;
            }
        }
    }
}

// `count` values from row[first] on, the rest `without`: 16 bytes a load, at any alignment, where there are four.
template <int V>
__device__ __forceinline__ void load_some(const float* row, int first, int count, float without, float (&out)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        if (i + 4 <= count) {
            float four[4];
            unpack<MOE_DTYPE_F32>(load_bytes<16>(row + first + i), four);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[i + j] = four[j];
        } else {
#pragma unroll
            for (int j = i; j < i + 4; ++j) out[j] = j < count ? row[first + j] : without;
        }
    }
}

// e^x by hardware exp2: within 1.224 |x| 2^-24 for the argument and 2^-23 of its own, of scores that order (which
// choose_fast counts), of weights and of gradients alike; 0 below 2^-126.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// A token's lanes are one wave, whose LDS accesses are in order: only the compiler has to keep it.
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The lane's best two of a group, then the group's, over group_lanes lanes (a power of two).
template <int LANES>
__device__ __forceinline__ void best_two(float& first, float& second, int group_lanes) {
    auto merge = [&](float f, float s) {
        second = fmaxf(fmaxf(second, s), fminf(first, f));
        first = fmaxf(first, f);
    };
    if (LANES >= 2 && group_lanes >= 2) merge(dpp_move<kDppXor1>(first), dpp_move<kDppXor1>(second));
    if (LANES >= 4 && group_lanes >= 4) merge(dpp_move<kDppXor2>(first), dpp_move<kDppXor2>(second));
    if (LANES >= 8 && group_lanes >= 8) merge(dpp_move<kDppHalfMirror>(first), dpp_move<kDppHalfMirror>(second));
    if (LANES >= 16 && group_lanes >= 16) merge(dpp_move<kDppMirror>(first), dpp_move<kDppMirror>(second));
    if (LANES >= 32 && group_lanes >= 32) merge(__shfl_xor(first, 16), __shfl_xor(second, 16));
}

// A float's bits as an unsigned integer of the same order; 0 stands for no key.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

// Orders the lane's keys, largest first, with their places (an odd-even merge network).
template <int V>
__device__ __forceinline__ void sort_keys(uint32_t (&key)[V], int (&place)[V]) {
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const int x = i + j, y = i + j + k;
                        const uint32_t kx = key[x], ky = key[y];
                        const int px = place[x], py = place[y];
                        const bool swap = ky > kx;
                        key[x] = swap ? ky : kx;
                        key[y] = swap ? kx : ky;
                        place[x] = swap ? py : px;
                        place[y] = swap ? px : py;
                    }
}

// Candidates whose order is worked out in 64 bits, a lane each.
constexpr int kCandidates = 16;

// Softmax's sum in 64 bits, relative to the token's largest logit. (Loops of few instructions, here and below: what
// only a token in a thousand comes to is not in the instruction cache.)
template <int LANES>
__device__ __forceinline__ double exact_total(const ScoreArgs& a, const Place& p, const float* row, float top) {
    double total = 0.0;
    if (a.sigmoid) return 1.0;
#pragma unroll 1
    for (int i = 0; i < p.count; ++i) total += exp(static_cast<double>(row[p.first + i]) - static_cast<double>(top));
#pragma unroll 1
    for (int d = 1; d < LANES; d <<= 1) total += lane_xor(total, d);
    return total;
}

// Expert id's score and bias in 64 bits.
__device__ __forceinline__ double exact_key(const ScoreArgs& a, const float* row, int id, float top, double total) {
    const double x = static_cast<double>(row[id]);
    const double e = exp(a.sigmoid ? -x : x - static_cast<double>(top));
    return (a.sigmoid ? 1.0 / (1.0 + e) : e / total) + (a.bias != nullptr ? static_cast<double>(a.bias[id]) : 0.0);
}

// Whether the lane's group takes part, by its exact score.
template <int LANES>
__device__ __forceinline__ bool exact_open(const ScoreArgs& a, const Place& p, const float* row, float top) {
    const double minus = -__builtin_inf();
    const double total = exact_total<LANES>(a, p, row, top);
    double first = minus, second = minus;
#pragma unroll 1
    for (int i = 0; i < p.count; ++i) {
        if (!(row[p.first + i] > -__builtin_inff())) continue;
        const double key = exact_key(a, row, p.first + i, top, total);
        second = most(second, key < first ? key : first);
        first = most(first, key);
    }
#pragma unroll 1
    for (int d = 1; d < p.group_lanes; d <<= 1) {
        const double f = lane_xor(first, d), s = lane_xor(second, d);
        second = most(most(second, s), f < first ? f : first);
        first = most(first, f);
    }
    const double group = a.group_best == 2 && second > minus ? first + second : first;
    const int mine = p.group;
    int before = 0;
#pragma unroll 1
    for (int o = p.group_lanes; o < LANES; o += p.group_lanes) {
        const double other = lane_xor(group, o);
        const int index = (p.lane ^ o) >> a.lane_shift;
        before += index < a.groups && (other > group || (other == group && index < mine));
    }
    return mine < a.groups && before < a.top_groups;
}

// Chooses by fp32 keys into picked[0..topk); true where that does not decide it. Where groups are too near each
// other to tell which take part, their scores are worked out in 64 bits; where keys are (or equal), among the chosen ones and
// those next to them, these candidates alone are ordered in 64 bits. `row`: the token's logits;
// `scores`: its room for a score a group; `exact`: for a key a candidate.
template <int LANES, int V>
__device__ __forceinline__ bool choose_fast(const ScoreArgs& a, const Place& p, const float* row, const float (&l)[V],
                                            const float (&b)[V], int* picked, float* scores, double* exact) {
    const bool has_bias = a.bias != nullptr;
    const float minus = -__builtin_inff();
    bool unsure = false;
    uint32_t key[V];
    float near = 0.0f, largest_logit = minus;
    if (!has_bias) {
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = l[i] > minus ? ordered(l[i]) : 0u;
    }
    if (has_bias || a.groups > 1) {
        float s[V];
        // How far the token's keys may be off, in units of u = 2^-24: `reach` from the scores, `weight` times the largest
        // bias. log2 e's own rounding and the product's put e^x's argument off by 1.224 |x| u (softmax's difference adds
        // |x| u), exp2 and a reciprocal are within 2 u.
        //  * sigmoid: s is off by s ((1 - s) (1.224 |l| + 2) + 3) u < s (4.01 + 1.5 L) u, L = max(-l, 0): what the
        //    argument's rounding does grows with the logit's size while s vanishes. A key adds (s + |b|) u. So two keys
        //    are off by 2 (s (5.01 + 1.5 L) + |b|), and two sums of two keys, with their roundings and the comparison's,
        //    by s (26.1 + 6 L) + 10 |b|: below 2 and 4.6 times max(s (8 + 2 L), 8 |b|). s (8 + 2 L) rises with l, so
        //    the token's largest logit has the most.
        //  * softmax: V + 5 for the sum's roundings, 11 for its terms (the mean of |x| weighted by e^x is below 4 with up to
        //    512 terms), 5 for exp, reciprocal and product, and 2.224 |x| e^x < 0.9 of the largest score: (V + 22) of that
        //    one. With key and sums as above below 2 and 4.6 times (V + 24) max(s, |b|).
        // Scores below the normal range are 0: off by 2^-126.
        float reach, weight;
        if (a.sigmoid) {
            float top = l[0];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[i] = __builtin_amdgcn_rcpf(1.0f + fast_exp(-l[i]));
                top = fmaxf(top, l[i]);
            }
            weight = 8.0f;
            reach = __builtin_amdgcn_rcpf(1.0f + fast_exp(-top)) * (8.0f + 2.0f * fminf(fmaxf(-top, 0.0f), 128.0f));
        } else {
            float top = l[0];
#pragma unroll
            for (int i = 1; i < V; ++i) top = fmaxf(top, l[i]);
            top = lanes_reduce<MaxOp, LANES>(top);
            largest_logit = top;
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[i] = fast_exp(l[i] - top);
                total += s[i];
            }
            const float inverse = __builtin_amdgcn_rcpf(lanes_reduce<SumOp, LANES>(total));
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] *= inverse;
            weight = V + 24;
            reach = weight * inverse;
        }
        // Magnitudes as integers: of numbers they order alike, and an infinity's or NaN's are the largest.
        uint32_t drawn = 0;
        float first = minus, second = minus;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool in = l[i] > minus;
            const float k = in ? s[i] + b[i] : minus;
            drawn = max(drawn, __float_as_uint(b[i]) & 0x7fffffffu);
            second = fmaxf(second, fminf(first, k));
            first = fmaxf(first, k);
            if (has_bias) key[i] = in ? ordered(k) : 0u;
        }
        const uint32_t size = lanes_max<LANES>(max(__float_as_uint(reach), __float_as_uint(weight * __uint_as_float(drawn))));
        near = 0x1p-23f * __uint_as_float(size) + 0x1p-124f;
        // A key that is no number, infinite, or so large that a sum of two is: the other path sorts that out.
        unsure = size >= 0x7e800000u;
        if (a.groups > 1) {
            best_two<LANES>(first, second, p.group_lanes);
            const float group = a.group_best == 2 && second > minus ? first + second : first;
            const int mine = p.group;
            // Lanes past the last group bring -inf, which is before and close to none.
            if ((p.lane & (p.group_lanes - 1)) == 0) scores[mine] = group;
            wave_fence();
            // Groups that are certainly before this one, and those that may be (itself among them).
            const float low = group - 2.3f * near, high = group + 2.3f * near;
            int before = 0, maybe = 0;
            const int places = LANES >> a.lane_shift;
            for (int g = 0; g < places; g += 4) {
                float other[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) other[j] = j < 2 || places > 2 ? scores[g + j] : minus;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    before += other[j] > high;
                    maybe += other[j] >= low;
                }
            }
            const bool real = mine < a.groups;
            // Only whether it is among the best counts; of groups without an expert left there is nothing to choose.
            bool open = real && before < a.top_groups;
            const bool cut = open && group > minus && maybe > a.top_groups;
            if constexpr (LANES < kCandidates) {
                unsure |= cut;
            } else if (__ballot(cut) != 0) {
                open = exact_open<LANES>(a, p, row, largest_logit);
            }
            if (!open) {
#pragma unroll
                for (int i = 0; i < V; ++i) key[i] = 0u;
            }
        }
    }
    int place[V];
#pragma unroll
    for (int i = 0; i < V; ++i) place[i] = p.first + i;
    sort_keys<V>(key, place);
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t segment = (LANES == 64 ? ~0ull : ((1ull << (LANES & 63)) - 1)) << (lane / LANES * LANES);
    const uint64_t lower = segment & ((1ull << lane) - 1);
    if (!has_bias) near = 0.0f;  // keys are the logits themselves
    float previous = __builtin_inff();
    bool close = false;
    // (Unrolled: after k + 1 choices at most kMaxTopk - k + 1 of a lane's keys are still looked at.)
#pragma unroll
    for (int k = 0; k < kMaxTopk; ++k) {
        if (k == a.topk) break;
        const uint32_t top = lanes_max<LANES>(key[0]);
        const uint64_t with = __ballot(key[0] == top);
        // The lowest lane that has it.
        const bool owner = LANES == 64 ? static_cast<int>(lane) == __builtin_ctzll(with)
                                       : key[0] == top && (with & lower) == 0;
        if (owner) {
            picked[k] = place[0];
#pragma unroll
            for (int i = 0; i < V && i <= kMaxTopk - k; ++i) {
                key[i] = i + 1 < V ? key[i + 1] : 0u;
                place[i] = i + 1 < V ? place[i + 1] : 0;
            }
        }
        const float value = unordered(top);
        close |= !(previous - value > near);  // neighbours in the order, equal ones included
        unsure |= top == 0u;                  // no expert left
        previous = value;
    }
    // Those left out that are as near to the last one chosen.
    auto next_near = [&](uint32_t next) { return next != 0u && !(previous - unordered(next) > near); };
    uint32_t next = lanes_max<LANES>(key[0]);
    close |= next_near(next);
    if constexpr (LANES < kCandidates) {
        return unsure || close;
    } else {
        bool part = close && (__ballot(unsure) & segment) == 0;  // of the token's lanes alike
        if (__ballot(part) == 0) return unsure;
        constexpr uint32_t kUnknown = ~0u;  // a second key of the lane's behind its last choice: not kept
        int count = a.topk;
        for (bool more = part;;) {
            more = more && next_near(next);
            if (more && (next == kUnknown || count == kCandidates)) {
                unsure = true;
                more = part = false;
            }
            const uint64_t with = __ballot(more && key[0] == next);
            if (with == 0) break;
            if (more && key[0] == next && (with & lower) == 0) {
                picked[count] = place[0];
                key[0] = key[1];
                place[0] = place[1];
                key[1] = kUnknown;
            }
            count += more;
            next = lanes_max<LANES>(key[0]);
        }
        const double total = has_bias ? exact_total<LANES>(a, p, row, largest_logit) : 1.0;
        wave_fence();
        part = part && p.lane < count;
        int id = 0, rank = 0;
        double mine = 0.0;
        if (part) {
            id = picked[p.lane];
            mine = has_bias ? exact_key(a, row, id, largest_logit, total) : static_cast<double>(row[id]);
            exact[p.lane] = mine;
        }
        wave_fence();
        for (int c = 0; c < kCandidates; c += 4) {
#pragma unroll
            for (int j = c; j < c + 4; ++j) {
                const double other = exact[j];
                rank += j < count && (other > mine || (other == mine && picked[j] < id));
            }
        }
        wave_fence();
        if (part && rank < a.topk) picked[rank] = id;
        return unsure;
    }
}

template <int LANES, int V>
__global__ __launch_bounds__(256) void route_scored_kernel(ScoreArgs a) {
    constexpr int TOKENS = 256 / LANES;
    constexpr int GROUPS = LANES < 64 ? LANES : 64;  // a lane each at least
    constexpr int ROOM = LANES < kCandidates ? kMaxTopk : kCandidates;
    __shared__ int picked[TOKENS][ROOM];
    __shared__ double exact[TOKENS][LANES < kCandidates ? 1 : kCandidates];
    __shared__ float scores[TOKENS][GROUPS];
    const int lane = threadIdx.x & 63;
    const int slot = threadIdx.x / LANES;  // the token's place in the workgroup: one wave's
    const int64_t token = static_cast<int64_t>(blockIdx.x) * TOKENS + slot;
    Place p;
    p.lane = lane % LANES;
    p.group_lanes = 1 << a.lane_shift;
    p.group = p.lane >> a.lane_shift;
    const int part = p.lane & (p.group_lanes - 1);
    p.first = p.group * a.group_size + part * V;
    p.count = p.group < a.groups ? max(0, min(V, a.group_size - part * V)) : 0;
    const bool live = token < a.tokens;
    if (!live) p.count = 0;  // these lanes take part in the reductions only
    float l[V], b[V];
    const float* row = a.logits + token * a.experts;
    load_some<V>(row, p.first, p.count, -__builtin_inff(), l);
    if (a.bias != nullptr) {
        load_some<V>(a.bias, p.first, p.count, 0.0f, b);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = 0.0f;
    }
    bool number = true;
#pragma unroll
    for (int i = 0; i < V; ++i) number &= l[i] == l[i];
    const uint64_t segment = (LANES == 64 ? ~0ull : ((1ull << (LANES & 63)) - 1)) << (lane / LANES * LANES);
    number = (__ballot(!number) & segment) == 0;
    const bool unsure = choose_fast<LANES, V>(a, p, row, l, b, picked[slot], scores[slot], exact[slot]) || !number;
    if (__ballot(unsure && live) != 0) {
        int rank[V];
        choose<LANES, V>(a, p, l, b, rank);
        wave_fence();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (rank[i] >= 0) picked[slot][rank[i]] = p.first + i;
    }
    wave_fence();

    // Weights: slot k on lane k, several a lane where the segment has fewer than eight. Renormalised ones from
    // scores relative to the largest chosen logit, so that scores too small for fp32 keep their ratio:
    // softmax e^(l - m); sigmoid e^(min(l, 0) - min(m, 0)) / (1 + e^-|l|).
    constexpr int WIDTH = LANES < kMaxTopk ? LANES : kMaxTopk, SLOTS = kMaxTopk / WIDTH;
    const float minus = -__builtin_inff();
    const bool all = !a.sigmoid && !a.renormalize;
    float top = minus, sum = 0.0f;
    if (all) {
#pragma unroll
        for (int i = 0; i < V; ++i) top = fmaxf(top, l[i]);
        top = lanes_reduce<MaxOp, LANES>(top);
#pragma unroll
        for (int i = 0; i < V; ++i) sum += l[i] > minus ? fast_exp(l[i] - top) : 0.0f;
        sum = lanes_reduce<SumOp, LANES>(sum);
    }
    int id[SLOTS];
    float chosen[SLOTS], w[SLOTS];
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        const int k = j * WIDTH + p.lane;
        const bool mine = live && p.lane < WIDTH && k < a.topk;
        id[j] = mine ? picked[slot][k] : -1;
        chosen[j] = mine ? row[id[j]] : minus;
        if (!all) top = fmaxf(top, chosen[j]);
    }
    if (!all) top = lanes_reduce<MaxOp, WIDTH>(top);
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        const float x = chosen[j];
        w[j] = 0.0f;
        if (x > minus) {
            if (!a.sigmoid)
                w[j] = fast_exp(x - top);
            else if (a.renormalize)
                w[j] = fast_exp(fminf(x, 0.0f) - fminf(top, 0.0f)) * __builtin_amdgcn_rcpf(1.0f + fast_exp(-fabsf(x)));
            else
                w[j] = __builtin_amdgcn_rcpf(1.0f + fast_exp(-x));
        }
        if (!all) sum += w[j];
    }
    if (!all) sum = lanes_reduce<SumOp, WIDTH>(sum);
    // Nothing but experts that are out: weights 0.
    float divisor = a.renormalize || !a.sigmoid ? (sum == 0.0f ? 1.0f : sum) : 1.0f;
    if (!number) divisor = __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < SLOTS; ++j)
        if (id[j] >= 0) {
            const int64_t at = token * a.topk + j * WIDTH + p.lane;
            a.ids[at] = id[j];
            a.weights[at] = w[j] / divisor * a.scale;
        }
}

template <int LANES, int V>
void run(ScoreArgs a, hipStream_t stream) {
    // (Divisions are the host's.)
    a.group_size = a.experts / a.groups;
    a.lane_shift = 0;
    while (V << a.lane_shift < a.group_size) ++a.lane_shift;
    const int64_t threads = a.tokens * LANES;
    route_scored_kernel<LANES, V><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, stream>>>(a);
}

template <int V>
void by_lanes(const ScoreArgs& a, int lanes, hipStream_t stream) {
    switch (lanes) {
        case 1: return run<1, V>(a, stream);
        case 2: return run<2, V>(a, stream);
        case 4: return run<4, V>(a, stream);
        case 8: return run<8, V>(a, stream);
        case 16: return run<16, V>(a, stream);
        case 32: return run<32, V>(a, stream);
        default: return run<64, V>(a, stream);
    }
}

int power_of_two(int n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

// Lanes of a token with v experts a lane: whole lanes a group, a power of two of them.
int lanes_of(const ScoreArgs& a, int v) {
    const int size = a.experts / a.groups;
    return power_of_two(a.groups) * power_of_two((size + v - 1) / v);
}

}  // namespace

int launch_route_scored(const ScoreArgs& a, hipStream_t stream) {
    // Four experts a lane where that fits a wave, else eight or sixteen. Eight as well for large batches of more than
    // 64 experts, where instructions count and not the length of a lane's chain: more tokens share a wave's
    // choices. Four against eight, top-8 by sigmoid and bias: 16384 tokens of 256 experts in 8 groups 17.5 and
    // 14.3 us, of 128 experts 9.4 and 8.4; 8192 of 64 in 8 groups 6.1 and 10.5; one of 256 4.2 and 4.7; 2048 of 128
    // in 8 groups 4.7 and 6.5.
    const bool large = a.tokens >= 4096 && a.experts > 64 && lanes_of(a, 8) <= kWave;
    if (!large && lanes_of(a, 4) <= kWave)
        by_lanes<4>(a, lanes_of(a, 4), stream);
    else if (lanes_of(a, 8) <= kWave)
        by_lanes<8>(a, lanes_of(a, 8), stream);
    else
        by_lanes<16>(a, lanes_of(a, 16), stream);
    return check_launch("route_scored");
}

// -- gradient ----------------------------------------------------------------
//
//   renormalised: t_j = scale (g_j - sum_i g_i w_i) / S, w the chosen scores over their sum S
//   dl = t s (1 - s) for chosen ones (sigmoid),  s (t - sum t s) for all (softmax)
//
// Renormalised softmax: dl_j = scale w_j (g_j - sum g w); renormalised sigmoid:
// dl_j = scale w_j (1 - s_j) (g_j - sum g w). Both need only the chosen logits.

namespace {

// LANES lanes a token, V experts of its row each. Slot k of the chosen ones is worked out by lane k alone
// (several by a lane where the segment has fewer than eight) and reaches the others through LDS.
template <int LANES, int V>
__global__ __launch_bounds__(256) void route_scored_grad_kernel(ScoreGradArgs a) {
    constexpr int TOKENS = 256 / LANES, WIDTH = LANES < kMaxTopk ? LANES : kMaxTopk, SLOTS = kMaxTopk / WIDTH;
    __shared__ int ids[TOKENS][kMaxTopk];
    __shared__ float grads[TOKENS][kMaxTopk];
    const int slot = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * TOKENS + slot;
    const int first = lane * V;
    const bool live = token < a.tokens;
    const int count = live ? max(0, min(V, a.experts - first)) : 0;
    const float* row = a.logits + token * a.experts;
    const float minus = -__builtin_inff();
    const bool dense = !a.sigmoid && !a.renormalize;
    int id[SLOTS];
    float chosen[SLOTS], g[SLOTS];
    float top = minus;
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        const int k = j * WIDTH + lane;
        const bool mine = live && lane < WIDTH && k < a.topk;
        id[j] = mine ? a.ids[token * a.topk + k] : -1;
        const bool in = id[j] >= 0 && id[j] < a.experts;
        chosen[j] = in ? row[id[j]] : minus;
        g[j] = in ? a.grad_weights[token * a.topk + k] : 0.0f;
        if (!dense) top = fmaxf(top, chosen[j]);
    }
    float l[V];
    float total = 0.0f;
    if (dense) {
        load_some<V>(row, first, count, minus, l);
#pragma unroll
        for (int i = 0; i < V; ++i) top = fmaxf(top, l[i]);
        top = lanes_reduce<MaxOp, LANES>(top);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            l[i] = l[i] == minus ? 0.0f : fast_exp(l[i] - top);
            total += l[i];
        }
        total = lanes_reduce<SumOp, LANES>(total);
        total = total == 0.0f ? 0.0f : 1.0f / total;
    } else {
        top = lanes_reduce<MaxOp, WIDTH>(top);
    }
    // Scores (relative to `top` where they are renormalised), and 1 - s of a sigmoid.
    float s[SLOTS], rest[SLOTS];
    float sum = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        const float x = chosen[j];
        rest[j] = 1.0f;
        s[j] = 0.0f;
        if (!(x == minus)) {
            if (a.sigmoid) {
                rest[j] = __builtin_amdgcn_rcpf(1.0f + fast_exp(x));
                s[j] = a.renormalize ? fast_exp(fminf(x, 0.0f) - fminf(top, 0.0f)) * __builtin_amdgcn_rcpf(1.0f + fast_exp(-fabsf(x)))
                                     : __builtin_amdgcn_rcpf(1.0f + fast_exp(-x));
            } else {
                s[j] = fast_exp(x - top) * (dense ? total : 1.0f);
            }
        }
        sum += s[j];
    }
    sum = lanes_reduce<SumOp, WIDTH>(sum);
    const float divisor = a.renormalize && sum != 0.0f ? sum : 1.0f;
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        s[j] /= divisor;  // one of a single chosen expert is exactly 1
        dot += s[j] * g[j];
    }
    dot = lanes_reduce<SumOp, WIDTH>(dot);
    const float mean = a.sigmoid && !a.renormalize ? 0.0f : dot;
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        const int k = j * WIDTH + lane;
        if (lane < WIDTH) {
            ids[slot][k] = id[j];
            grads[slot][k] = a.scale * s[j] * rest[j] * (dense ? g[j] : g[j] - mean);
        }
    }
    wave_fence();
    if constexpr (LANES > WIDTH) dot = __shfl(dot, 0, LANES);  // the lanes without slots
    float out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = dense ? -(l[i] * total) * dot * a.scale : 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxTopk; ++k) {
        const int at = ids[slot][k] - first;
        const float d = grads[slot][k];
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] += at == i ? d : 0.0f;
    }
    float* to = a.grad_logits + token * a.experts + first;
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        if (i + 4 <= count) {
            const float four[4] = {out[i], out[i + 1], out[i + 2], out[i + 3]};
            store_bytes<16>(to + i, pack<MOE_DTYPE_F32>(four));
        } else {
#pragma unroll
            for (int j = i; j < i + 4; ++j)
                if (j < count) to[j] = out[j];
        }
    }
}

template <int LANES, int V>
void run_grad(const ScoreGradArgs& a, hipStream_t stream) {
    const int64_t threads = a.tokens * LANES;
    route_scored_grad_kernel<LANES, V><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, stream>>>(a);
}

}  // namespace

int launch_route_scored_backward(const ScoreGradArgs& a, hipStream_t stream) {
    switch (power_of_two((a.experts + 3) / 4)) {
        case 1: run_grad<1, 4>(a, stream); break;
        case 2: run_grad<2, 4>(a, stream); break;
        case 4: run_grad<4, 4>(a, stream); break;
        case 8: run_grad<8, 4>(a, stream); break;
        case 16: run_grad<16, 4>(a, stream); break;
        case 32: run_grad<32, 4>(a, stream); break;
        case 64: run_grad<64, 4>(a, stream); break;
        default: run_grad<64, 8>(a, stream); break;
    }
    return check_launch("route_scored_backward");
}

}  // namespace moe
