// Routing by scores: softmax or sigmoid of the logits, a bias that only takes part in the
// choice, groups of experts, top-k, renormalised and scaled weights; and its gradient.
//
//   s = sigmoid(l) or softmax(l);  key = s + bias, or without a bias the logit itself
//   (the same order);  a group's score: the sum of its best one or two s + bias;
//   the best groups, the best keys in them, ties to the lowest index;
//   w = scale s_j / sum_chosen s  or  scale s_j.
//
// A token is a segment of LANES lanes of a wave, V experts a lane, every group in lanes of
// its own. The choice is by exact value: scores are fp32 first, and a token whose order
// hangs on a difference within their rounding is decided again with fp64 scores by its
// wave, so that the ids are the definition's and do not depend on how exp rounds.
#include "row_ops.h"

namespace moe {

namespace {

template <int CTRL>
__device__ __forceinline__ double dpp_move(double x) {
    const uint64_t u = __double_as_longlong(x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xf, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xf, 0xf, true);
    return __longlong_as_double(static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ float lane_xor(float x, int mask) { return __shfl_xor(x, mask); }
__device__ __forceinline__ double lane_xor(double x, int mask) { return __shfl_xor(x, mask); }

__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }

// The largest over aligned segments of `lanes` lanes, in each lane.
template <int LANES>
__device__ __forceinline__ float segment_max(float x) {
    return lanes_reduce<MaxOp, LANES>(x);
}
template <int LANES>
__device__ __forceinline__ double segment_max(double x) {
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) x = most(x, lane_xor(x, d));
    return x;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

template <typename F> __device__ __forceinline__ F minus_inf();
template <> __device__ __forceinline__ float minus_inf<float>() { return -__builtin_inff(); }
template <> __device__ __forceinline__ double minus_inf<double>() { return -__builtin_inf(); }

// Where a lane's V experts lie.
struct Place {
    int first;   // the lane's first expert
    int count;   // its experts (0: none)
    int lane;    // lane of the token's segment
    int group_lanes;
};

// Chooses the token's experts by keys of type F: rank[i] = the slot of the lane's expert i
// or -1. Returns whether the order hangs on a difference of at most `doubt` times the
// largest key (fp32's rounding; 0 in fp64).
template <typename F, int LANES, int V>
__device__ __forceinline__ bool choose(const ScoreArgs& a, const Place& p, const float (&l)[V], const float (&b)[V],
                                       F doubt, int (&rank)[V]) {
    const bool has_bias = a.bias != nullptr;
    F key[V], score[V];
    F largest = 0;
    if (has_bias || a.groups > 1) {
        if (a.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; ++i) score[i] = F(1) / (F(1) + exp_of(-static_cast<F>(l[i])));
        } else {
            F top = minus_inf<F>();
#pragma unroll
            for (int i = 0; i < V; ++i) top = most(top, static_cast<F>(l[i]));
            top = segment_max<LANES>(top);
            F total = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                score[i] = l[i] == -__builtin_inff() ? F(0) : exp_of(static_cast<F>(l[i]) - top);
                total += score[i];
            }
#pragma unroll
            for (int d = 1; d < LANES; d <<= 1) total += lane_xor(total, d);
#pragma unroll
            for (int i = 0; i < V; ++i) score[i] /= total;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            score[i] += static_cast<F>(b[i]);
            // An expert that is out (a logit of -inf, or no number) has no key.
            if (!(l[i] > -__builtin_inff()) || !(score[i] == score[i])) score[i] = minus_inf<F>();
            if (score[i] > minus_inf<F>()) largest = most(largest, most(most(score[i], -score[i]), most(static_cast<F>(b[i]), static_cast<F>(-b[i]))));
        }
        largest = segment_max<LANES>(largest);
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        key[i] = has_bias ? score[i] : (l[i] > -__builtin_inff() ? static_cast<F>(l[i]) : minus_inf<F>());
    // Keys of a bias are rounded; logits are what they are.
    const F near = doubt * largest;
    bool unsure = false;
    bool open = true;
    if (a.groups > 1) {
        // The lane's best two, then the group's.
        F first = minus_inf<F>(), second = minus_inf<F>();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < p.count) {
                second = most(second, score[i] < first ? score[i] : first);
                first = most(first, score[i]);
            }
        for (int d = 1; d < p.group_lanes; d <<= 1) {
            const F f = lane_xor(first, d), s = lane_xor(second, d);
            second = most(most(second, s), f < first ? f : first);
            first = most(first, f);
        }
        F group = first;
        if (a.group_best == 2 && second > minus_inf<F>()) group += second;
        // Its place among the groups, ties to the lower one; lanes without a group are last.
        const int mine = p.lane / p.group_lanes;
        const bool real = mine < a.groups;
        int before = 0;
        for (int o = 1; o < LANES / p.group_lanes; ++o) {
            const F other = lane_xor(group, o * p.group_lanes);
            const int index = mine ^ o;
            if (index < a.groups && (other > group || (other == group && index < mine))) ++before;
            const F gap = other > group ? other - group : group - other;
            unsure |= real && index < a.groups && gap <= 4 * near;
        }
        open = real && before < a.top_groups;
    }
    // Chosen experts hold no key any more; those that have none in an open group are
    // chosen last, in order, with the key below every other.
    uint32_t left = 0;  // experts of the lane that can be chosen
#pragma unroll
    for (int i = 0; i < V; ++i) {
        rank[i] = -1;
        if (open && i < p.count) left |= 1u << i;
        if (!open || i >= p.count) key[i] = minus_inf<F>();
    }
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t segment = (LANES == 64 ? ~0ull : ((1ull << (LANES & 63)) - 1)) << (lane / LANES * LANES);
    F previous = 0;
    for (int k = 0; k <= a.topk; ++k) {
        F best = minus_inf<F>();
#pragma unroll
        for (int i = 0; i < V; ++i) best = most(best, key[i]);
        const F top = segment_max<LANES>(best);
        // The order of neighbours, the first one left out among them.
        if (has_bias && k > 0) unsure |= previous > minus_inf<F>() && top > minus_inf<F>() && previous - top <= 2 * near;
        previous = top;
        if (k == a.topk) break;
        const uint64_t with = __ballot(left != 0 && best == top) & segment;
        const bool owner = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(with >> 32),
                                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(with), 0)) == 0 &&
                           (with >> lane & 1);
        if (owner) {
            bool done = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool take = !done && (left >> i & 1) && key[i] == top;
                rank[i] = take ? k : rank[i];
                key[i] = take ? minus_inf<F>() : key[i];
                left &= take ? ~(1u << i) : ~0u;
                done |= take;
            }
        }
    }
    return unsure;
}

template <int LANES, int V>
__global__ __launch_bounds__(256) void route_scored_kernel(ScoreArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t token = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LANES;
    Place p;
    p.lane = lane % LANES;
    const int size = a.experts / a.groups;
    const int per = (size + V - 1) / V;
    p.group_lanes = per <= 1 ? 1 : 1 << (32 - __builtin_clz(per - 1));
    const int group = p.lane / p.group_lanes, part = p.lane % p.group_lanes;
    p.first = group * size + part * V;
    p.count = group < a.groups ? max(0, min(V, size - part * V)) : 0;
    if (token >= a.tokens) p.count = 0;  // these lanes take part in the reductions only
    float l[V], b[V];
    const float* row = a.logits + token * a.experts + p.first;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        l[i] = i < p.count ? row[i] : -__builtin_inff();
        b[i] = i < p.count && a.bias != nullptr ? a.bias[p.first + i] : 0.0f;
    }
    int rank[V];
    // A score is within 14 roundings of 2^-24 (exp's argument and value, a sum of at most 16
    // and 6 levels, a division), its key 15 of the largest key or bias: 2^-20 of that.
    const bool unsure = choose<float, LANES, V>(a, p, l, b, 0x1p-20f, rank);
    if (__ballot(unsure && token < a.tokens) != 0) choose<double, LANES, V>(a, p, l, b, 0.0, rank);
    if (token >= a.tokens) return;

    // Weights. Renormalised ones from scores relative to the largest chosen logit, so that
    // scores too small for fp32 keep their ratio: softmax e^(l - m); sigmoid
    // e^(min(l, 0) - min(m, 0)) / (1 + e^-|l|).
    bool number = true;
    float top = -__builtin_inff(), top_all = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        number &= l[i] == l[i];
        top_all = fmaxf(top_all, l[i]);
        if (rank[i] >= 0) top = fmaxf(top, l[i]);
    }
    const uint64_t segment = (LANES == 64 ? ~0ull : ((1ull << (LANES & 63)) - 1)) << (lane / LANES * LANES);
    number = (__ballot(!number) & segment) == 0;
    const bool all = !a.sigmoid && !a.renormalize;
    top = lanes_reduce<MaxOp, LANES>(all ? top_all : top);
    float w[V];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float s = 0.0f;
        if (l[i] > -__builtin_inff()) {
            if (!a.sigmoid)
                s = expf(l[i] - top);
            else if (a.renormalize)
                s = expf(fminf(l[i], 0.0f) - fminf(top, 0.0f)) / (1.0f + expf(-fabsf(l[i])));
            else
                s = 1.0f / (1.0f + expf(-l[i]));
        }
        w[i] = s;
        if (all || rank[i] >= 0) sum += s;
    }
    sum = lanes_reduce<SumOp, LANES>(sum);
    // Nothing but experts that are out: weights 0.
    float divisor = a.renormalize || !a.sigmoid ? (sum == 0.0f ? 1.0f : sum) : 1.0f;
    if (!number) divisor = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (rank[i] >= 0) {
            a.ids[token * a.topk + rank[i]] = p.first + i;
            a.weights[token * a.topk + rank[i]] = w[i] / divisor * a.scale;
        }
}

template <int LANES, int V>
void run(const ScoreArgs& a, hipStream_t stream) {
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
    // Four experts a lane where that fits a wave, else eight or sixteen.
    if (lanes_of(a, 4) <= kWave)
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

// LANES lanes a token, V experts of its row each.
template <int LANES, int V>
__global__ __launch_bounds__(256) void route_scored_grad_kernel(ScoreGradArgs a) {
    const int64_t token = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LANES;
    const int first = (threadIdx.x % LANES) * V;
    const bool live = token < a.tokens;
    const int count = live ? max(0, min(V, a.experts - first)) : 0;
    const float* row = a.logits + token * a.experts;
    const float minus = -__builtin_inff();
    const bool dense = !a.sigmoid && !a.renormalize;
    float l[V];
    float top = minus, total = 0.0f;
    if (dense) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            l[i] = i < count ? row[first + i] : minus;
            top = fmaxf(top, l[i]);
        }
        top = lanes_reduce<MaxOp, LANES>(top);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            l[i] = l[i] == minus ? 0.0f : expf(l[i] - top);
            total += l[i];
        }
        total = lanes_reduce<SumOp, LANES>(total);
        total = total == 0.0f ? 0.0f : 1.0f / total;
    }
    if (!live) return;
    int id[kMaxTopk];
    float chosen[kMaxTopk], g[kMaxTopk];
#pragma unroll
    for (int k = 0; k < kMaxTopk; ++k) {
        id[k] = k < a.topk ? a.ids[token * a.topk + k] : -1;
        const bool in = id[k] >= 0 && id[k] < a.experts;
        chosen[k] = in ? row[id[k]] : minus;
        g[k] = in ? a.grad_weights[token * a.topk + k] : 0.0f;
    }
    if (!dense) {
#pragma unroll
        for (int k = 0; k < kMaxTopk; ++k) top = fmaxf(top, chosen[k]);
    }
    // Scores (relative to `top` where they are renormalised), and 1 - s of a sigmoid.
    float s[kMaxTopk], rest[kMaxTopk];
    float sum = 0.0f, dot = 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxTopk; ++k) {
        rest[k] = 1.0f;
        s[k] = 0.0f;
        if (!(chosen[k] == minus)) {
            if (a.sigmoid) {
                rest[k] = 1.0f / (1.0f + expf(chosen[k]));
                s[k] = a.renormalize ? expf(fminf(chosen[k], 0.0f) - fminf(top, 0.0f)) / (1.0f + expf(-fabsf(chosen[k])))
                                     : 1.0f / (1.0f + expf(-chosen[k]));
            } else {
                s[k] = expf(chosen[k] - top) * (dense ? total : 1.0f);
            }
        }
        sum += s[k];
    }
    const float divisor = a.renormalize && sum != 0.0f ? sum : 1.0f;
#pragma unroll
    for (int k = 0; k < kMaxTopk; ++k) {
        s[k] /= divisor;  // one of a single chosen expert is exactly 1
        dot += s[k] * g[k];
    }
    const float mean = a.sigmoid && !a.renormalize ? 0.0f : dot;
    float out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = dense ? -(l[i] * total) * mean * a.scale : 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxTopk; ++k) {
        const float d = a.scale * s[k] * rest[k] * (dense ? g[k] : g[k] - mean);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] += id[k] == first + i ? d : 0.0f;
    }
    float* to = a.grad_logits + token * a.experts + first;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < count) to[i] = out[i];
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
