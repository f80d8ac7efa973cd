// The router of a mixture-of-experts layer: scores, group-limited top-k and route weights, the balance loss over sequences with its
// per-expert counts, and the logits' gradient of both.
//
// With z a token's logits (fp32; -inf: the expert is out of service) and s = 1 / (1 + exp(-z)):
//   key      softmax: z;  sigmoid: fl(s + bias), bias for the choice alone
//   groups   E / G consecutive experts each; a group's score is its largest key (softmax) or the sum of its two largest (sigmoid); the experts
//            of the best groups stay
//   choice   the K largest keys in descending order, ties to the lowest index, -1 where fewer than K are left
//   weights  softmax: over the row, normalised: over the chosen;  sigmoid: s, normalised: s / (sum of the chosen s + 1e-20);  times scale
// A wave holds a token's row, expert lane * V + v in register v of a lane.
#include <algorithm>
#include <type_traits>

#include "common.h"

#pragma clang fp contract(off)

namespace dpep {
namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr float kTiny = 1e-20f;  // keeps the sum of chosen sigmoids off zero (all of them underflow below a logit of -88)
constexpr int kRouterThreads = 256;
constexpr int kRouterWaves = kRouterThreads / kWave;
constexpr int kMaxRouterExperts = 1024;

template <int kType>
__device__ __forceinline__ float load_logit(const void* p, size_t i)
{
    if constexpr (kType == DPEP_TYPE_F32) return static_cast<const float*>(p)[i];
    if constexpr (kType == DPEP_TYPE_BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    return f16_to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <int kType>
__device__ __forceinline__ void store_logit(void* p, size_t i, float v)
{
    if constexpr (kType == DPEP_TYPE_F32) static_cast<float*>(p)[i] = v;
    if constexpr (kType == DPEP_TYPE_BF16) static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(f32_to_bf16(v));
    if constexpr (kType == DPEP_TYPE_F16) static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(pack_f16x2(v, 0.0f) & 0xffffu);
}
__device__ __forceinline__ int load_index(const void* p, bool wide, size_t i, int experts)
{
    const long long e = wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
    return e >= 0 && e < experts ? static_cast<int>(e) : -1;
}

// (The choice compares keys, so a key has to be the same 32 bits whoever computes it: IEEE divide and the library's exp.)
__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }

__device__ __forceinline__ float wave_max(float v)
{
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ float wave_sum(float v)
{
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// What the wave's lanes stored to LDS is there for all of them.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct Route {
    const void* logits;
    const float* bias;
    const uint8_t* token_mask;
    void* topk_idx;
    float* topk_weights;
    int tokens, experts, topk, groups, topk_groups;
    bool normalize, wide;
    float scale;
};

// Keeps the experts of the best groups: every other key becomes -inf.  keys_lds: the row's keys; groups_lds: a group's score each.
template <int V, bool kSigmoid>
__device__ void limit_groups(float (&key)[V], const Route& r, float* keys_lds, float* groups_lds, int lane)
{
    const int width = r.experts / r.groups;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (lane * V + v < r.experts) keys_lds[lane * V + v] = key[v];
    wave_sync();
    for (int g = lane; g < r.groups; g += kWave) {
        float first = -kInf, second = -kInf;
        for (int j = 0; j < width; ++j) {
            const float k = keys_lds[g * width + j];
            second = fmaxf(second, fminf(first, k));
            first = fmaxf(first, k);
        }
        groups_lds[g] = !kSigmoid || second == -kInf ? first : first + second;
    }
    wave_sync();
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = lane * V + v;
        if (e >= r.experts) continue;
        const int g = e / width;
        const float mine = groups_lds[g];
        int ahead = 0;
        for (int o = 0; o < r.groups; ++o) {
            const float other = groups_lds[o];
            ahead += other > mine || (other == mine && o < g);
        }
        if (ahead >= r.topk_groups) key[v] = -kInf;
    }
}

template <int V, int kType, bool kSigmoid>
__global__ __launch_bounds__(kRouterThreads) void route_kernel(const Route r)
{
    __shared__ float keys_lds[kRouterWaves][kWave * V];
    __shared__ float groups_lds[kRouterWaves][kWave * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int token = blockIdx.x * kRouterWaves + wave;
    if (token >= r.tokens) return;
    const size_t row = static_cast<size_t>(token) * r.experts;
    const bool real = r.token_mask == nullptr || r.token_mask[token] != 0;
    float key[V], z[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = lane * V + v;
        z[v] = e < r.experts ? load_logit<kType>(r.logits, row + e) : -kInf;
        float k = z[v];
        if constexpr (kSigmoid) {
            k = sigmoid(z[v]);
            if (r.bias != nullptr && e < r.experts) k += r.bias[e];
        }
        // a NaN ranks with +inf, so that it is chosen and shows in the weights; what is out of service ranks nowhere
        key[v] = z[v] == -kInf || !real ? -kInf : fminf(k, kInf);
    }
    float top = -kInf, total = 0.0f;
    if (!kSigmoid && !r.normalize) {
#pragma unroll
        for (int v = 0; v < V; ++v) top = fmaxf(top, z[v]);
        top = wave_max(top);
#pragma unroll
        for (int v = 0; v < V; ++v) total += z[v] == -kInf ? 0.0f : expf(z[v] - top);
        total = wave_sum(total);
    }
    if (r.groups > 1) limit_groups<V, kSigmoid>(key, r, keys_lds[wave], groups_lds[wave], lane);

    int mine = -1;  // lane k: the expert of slot k
    for (int k = 0; k < r.topk; ++k) {
        float best = key[0];
#pragma unroll
        for (int v = 1; v < V; ++v) best = fmaxf(best, key[v]);
        best = wave_max(best);
        if (best == -kInf) break;
        int at = 0x7fffffff;
#pragma unroll
        for (int v = V - 1; v >= 0; --v)
            if (key[v] == best) at = lane * V + v;
        for (int d = 32; d > 0; d >>= 1) at = min(at, __shfl_xor(at, d));
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (lane * V + v == at) key[v] = -kInf;
        if (lane == k) mine = at;
    }

    float weight = 0.0f;
    const float chosen = mine >= 0 ? load_logit<kType>(r.logits, row + mine) : -kInf;
    if constexpr (kSigmoid) {
        weight = mine >= 0 ? sigmoid(chosen) : 0.0f;
        if (r.normalize) weight = weight / (wave_sum(weight) + kTiny);
    } else {
        if (r.normalize) top = wave_max(chosen);
        weight = mine >= 0 ? expf(chosen - top) : 0.0f;
        if (r.normalize) total = wave_sum(weight);
        weight = mine >= 0 ? weight / total : 0.0f;
    }
    if (lane < r.topk) {
        const size_t to = static_cast<size_t>(token) * r.topk + lane;
        if (r.wide) static_cast<int64_t*>(r.topk_idx)[to] = mine;
        else static_cast<int32_t*>(r.topk_idx)[to] = mine;
        r.topk_weights[to] = weight * r.scale;
    }
}

// ---- balance loss ------------------------------------------------------------------------------------------------------------------
// Sequence b of N tokens with a route and R routes, c_e of them to expert e; p a token's softmax, or its sigmoids over their sum:
//   f_e = E c_e / R,  loss_b = sum_e f_e (sum_t p_te) / N
// Chunks of tokens leave one row of sums for every sequence they touch; (chunk + sequence) numbers these rows without a gap to spare.
struct Balance {
    const void* logits;
    const void* topk_idx;
    const int32_t* offsets;  // [sequences + 1], or null: one sequence
    int tokens, experts, topk, sequences, chunk, chunks;
    bool wide;
    float* sums;             // [chunks + sequences][experts]
    int32_t* counts;         // the same
    int32_t* members;        // [chunks + sequences]
};

__device__ __forceinline__ int sequence_begin(const int32_t* offsets, int b, int sequences, int tokens)
{
    if (offsets == nullptr) return b == 0 ? 0 : tokens;
    return min(max(offsets[b], 0), tokens);
}
// The last sequence that begins at `token` or in front of it.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int sequences, int token)
{
    if (offsets == nullptr) return 0;
    int low = 0, high = sequences;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (offsets[mid] <= token) low = mid;
        else high = mid;
    }
    return low;
}

// A row's probabilities; false for padding.  (1 / the sum of sigmoids for the gradient.)
template <int V, int kType, bool kSigmoid>
__device__ __forceinline__ void row_probabilities(const void* logits, size_t row, int experts, int lane, float (&p)[V], float (&s)[V], float& inverse)
{
    float z[V], top = -kInf, total = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = lane * V + v;
        z[v] = e < experts ? load_logit<kType>(logits, row + e) : -kInf;
        top = fmaxf(top, z[v]);
    }
    if constexpr (!kSigmoid) top = wave_max(top);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        s[v] = z[v] == -kInf ? 0.0f : kSigmoid ? sigmoid(z[v]) : expf(z[v] - top);
        total += s[v];
    }
    total = wave_sum(total);
    inverse = kSigmoid ? 1.0f / (total + kTiny) : total > 0.0f || total != total ? 1.0f / total : 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        p[v] = s[v] * inverse;
        if constexpr (kSigmoid) s[v] = z[v] == -kInf ? 0.0f : s[v] * sigmoid(-z[v]);  // ds/dz (1 - s would cancel)
    }
}

template <int V, int kType, bool kSigmoid>
__global__ __launch_bounds__(kRouterThreads) void balance_sums_kernel(const Balance c)
{
    __shared__ int counts[kWave * V];
    __shared__ float sums[kRouterWaves][kWave * V];
    __shared__ int members[kRouterWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int first = blockIdx.x * c.chunk, last = min(first + c.chunk, c.tokens);
    int begin = first;
    for (int b = sequence_of(c.offsets, c.sequences, first); b < c.sequences && begin < last; ++b) {
        const int end = b + 1 == c.sequences ? last : min(last, sequence_begin(c.offsets, b + 1, c.sequences, c.tokens));
        if (end <= begin) continue;
        for (int e = threadIdx.x; e < c.experts; e += kRouterThreads) counts[e] = 0;
        __syncthreads();
        float acc[V] = {};
        int held = 0;
        for (int t = begin + wave; t < end; t += kRouterWaves) {
            const int e = lane < c.topk ? load_index(c.topk_idx, c.wide, static_cast<size_t>(t) * c.topk + lane, c.experts) : -1;
            if (__ballot(e >= 0) == 0) continue;
            if (e >= 0) atomicAdd(&counts[e], 1);
            ++held;
            float p[V], s[V], inverse;
            row_probabilities<V, kType, kSigmoid>(c.logits, static_cast<size_t>(t) * c.experts, c.experts, lane, p, s, inverse);
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] += p[v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) sums[wave][lane * V + v] = acc[v];
        if (lane == 0) members[wave] = held;
        __syncthreads();
        const size_t slot = blockIdx.x + b;
        for (int e = threadIdx.x; e < c.experts; e += kRouterThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kRouterWaves; ++w) sum += sums[w][e];
            c.sums[slot * c.experts + e] = sum;
            c.counts[slot * c.experts + e] = counts[e];
        }
        if (threadIdx.x == 0) {
            int total = 0;
            for (int w = 0; w < kRouterWaves; ++w) total += members[w];
            c.members[slot] = total;
        }
        __syncthreads();
        begin = end;
    }
}

constexpr int kFinishThreads = 1024;
__global__ __launch_bounds__(kFinishThreads) void balance_finish_kernel(const Balance c, float* losses, int32_t* counts, int32_t* members)
{
    __shared__ float part[kFinishThreads / kWave];
    __shared__ int routes[kFinishThreads / kWave];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int begin = sequence_begin(c.offsets, b, c.sequences, c.tokens);
    const int end = b + 1 == c.sequences ? c.tokens : sequence_begin(c.offsets, b + 1, c.sequences, c.tokens);
    const int first = begin / max(c.chunk, 1), last = end > begin ? (end - 1) / c.chunk : first - 1;
    const int e = threadIdx.x;
    float sum = 0.0f;
    int count = 0;
    if (e < c.experts) {
        for (int i = first; i <= last; ++i) {
            sum += c.sums[static_cast<size_t>(i + b) * c.experts + e];
            count += c.counts[static_cast<size_t>(i + b) * c.experts + e];
        }
        counts[static_cast<size_t>(b) * c.experts + e] = count;
    }
    float product = wave_sum(sum * static_cast<float>(count));
    int total = count;
    for (int d = 32; d > 0; d >>= 1) total += __shfl_xor(total, d);
    if (lane == 0) {
        part[wave] = product;
        routes[wave] = total;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int held = 0;
        for (int i = first; i <= last; ++i) held += c.members[i + b];
        product = 0.0f;
        total = 0;
        for (int w = 0; w < kFinishThreads / kWave; ++w) {
            product += part[w];
            total += routes[w];
        }
        losses[b] = held > 0 ? product / static_cast<float>(held) * (static_cast<float>(c.experts) / static_cast<float>(total)) : 0.0f;
        members[b] = held;
    }
}

// ---- gradient of the logits --------------------------------------------------------------------------------------------------------
struct Backward {
    const void* logits;
    const void* topk_idx;
    const float* topk_weights;
    const float* grad_weights;  // null: no gradient comes through the route weights
    const int32_t* offsets;
    const int32_t* counts;      // [sequences][experts]; null: none comes through the balance loss
    const int32_t* members;
    const float* grad_losses;
    void* grad_logits;
    int tokens, experts, topk, sequences;
    bool normalize, wide;
    float scale;
};

template <int V, int kType, bool kSigmoid>
__global__ __launch_bounds__(kRouterThreads) void router_backward_kernel(const Backward c)
{
    __shared__ float rows[kRouterWaves][kWave * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int token = blockIdx.x * kRouterWaves + wave;
    if (token >= c.tokens) return;
    const size_t row = static_cast<size_t>(token) * c.experts, slot = static_cast<size_t>(token) * c.topk + lane;
    const int e = lane < c.topk ? load_index(c.topk_idx, c.wide, slot, c.experts) : -1;
    const bool padding = __ballot(e >= 0) == 0;
    float grad[V] = {};
    const bool dense = c.grad_weights != nullptr && !kSigmoid && !c.normalize;
    float p[V], s[V], inverse = 0.0f;
    if (!padding && (dense || c.counts != nullptr))
        row_probabilities<V, kType, kSigmoid>(c.logits, row, c.experts, lane, p, s, inverse);
    if (!padding && c.counts != nullptr) {
        // softmax: a p (f - sum f p); sigmoid: a s (1 - s) / sum s (f - sum f p);  a = grad / N
        const int b = sequence_of(c.offsets, c.sequences, token);
        float f[V], mean = 0.0f;
        int routes = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = lane * V + v;
            const int count = at < c.experts ? c.counts[static_cast<size_t>(b) * c.experts + at] : 0;
            routes += count;
            f[v] = static_cast<float>(count);
        }
        for (int d = 32; d > 0; d >>= 1) routes += __shfl_xor(routes, d);
        const float unit = routes > 0 ? static_cast<float>(c.experts) / static_cast<float>(routes) : 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            f[v] *= unit;
            mean += f[v] * p[v];
        }
        mean = wave_sum(mean);
        const float a = c.grad_losses[b] / static_cast<float>(max(c.members[b], 1));
#pragma unroll
        for (int v = 0; v < V; ++v) grad[v] = a * (f[v] - mean) * (kSigmoid ? s[v] * inverse : p[v]);
    }
    if (c.grad_weights != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) rows[wave][lane * V + v] = 0.0f;
        wave_sync();
        float g = e >= 0 ? c.grad_weights[slot] * c.scale : 0.0f, through = 0.0f;
        if (c.normalize) {
            const float w = e >= 0 ? c.topk_weights[slot] / c.scale : 0.0f;
            const float inner = wave_sum(g * w);
            g = e >= 0 ? g - inner : 0.0f;
            through = w * g;
        }
        if constexpr (kSigmoid) {
            const float z = e >= 0 ? load_logit<kType>(c.logits, row + e) : 0.0f;
            const float score = e >= 0 ? sigmoid(z) : 0.0f;
            through = g * score * sigmoid(-z);
            if (c.normalize) through = through / (wave_sum(score) + kTiny);
        }
        if (dense) {
            // p_e ([e chosen] g_e - sum_j g_j p_j)
            if (e >= 0) atomicAdd(&rows[wave][e], g);
            wave_sync();
            float inner = 0.0f, own[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                own[v] = rows[wave][lane * V + v];
                inner += padding ? 0.0f : own[v] * p[v];
            }
            inner = wave_sum(inner);
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (!padding) grad[v] += p[v] * (own[v] - inner);
        } else {
            if (e >= 0) atomicAdd(&rows[wave][e], through);
            wave_sync();
#pragma unroll
            for (int v = 0; v < V; ++v) grad[v] += rows[wave][lane * V + v];
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (lane * V + v < c.experts) store_logit<kType>(c.grad_logits, row + lane * V + v, grad[v]);
}

// ---- launches ----------------------------------------------------------------------------------------------------------------------
// Calls f with the registers per lane, the logits' type and the score as constants.
template <class F>
void with_variant(const dpep_router* r, F&& f)
{
    auto by_score = [&](auto v, auto type) {
        if (r->score == DPEP_SCORE_SIGMOID) f(v, type, std::integral_constant<bool, true>{});
        else f(v, type, std::integral_constant<bool, false>{});
    };
    auto by_type = [&](auto v) {
        if (r->logits_type == DPEP_TYPE_F32) by_score(v, std::integral_constant<int, DPEP_TYPE_F32>{});
        else if (r->logits_type == DPEP_TYPE_BF16) by_score(v, std::integral_constant<int, DPEP_TYPE_BF16>{});
        else by_score(v, std::integral_constant<int, DPEP_TYPE_F16>{});
    };
    const int lanes = (r->num_experts + kWave - 1) / kWave;
    if (lanes <= 1) by_type(std::integral_constant<int, 1>{});
    else if (lanes <= 2) by_type(std::integral_constant<int, 2>{});
    else if (lanes <= 4) by_type(std::integral_constant<int, 4>{});
    else if (lanes <= 8) by_type(std::integral_constant<int, 8>{});
    else by_type(std::integral_constant<int, 16>{});
}

int balance_chunk(int tokens) { return std::max(64, (tokens + 511) / 512); }

int check_router(const dpep_router* r, int num_tokens, const char* what)
{
    DPEP_REQUIRE(r != nullptr, "%s: router is NULL", what);
    DPEP_REQUIRE(num_tokens >= 0, "%s: num_tokens=%d", what, num_tokens);
    DPEP_REQUIRE(r->num_experts >= 1 && r->num_experts <= kMaxRouterExperts, "%s: num_experts=%d is not in [1, %d]", what, r->num_experts, kMaxRouterExperts);
    DPEP_REQUIRE(r->num_topk >= 1 && r->num_topk <= DPEP_MAX_TOPK && r->num_topk <= r->num_experts, "%s: num_topk=%d is not in [1, min(%d, num_experts)]", what,
                 r->num_topk, DPEP_MAX_TOPK);
    DPEP_REQUIRE(r->num_groups >= 1 && r->num_experts % r->num_groups == 0, "%s: num_groups=%d does not divide num_experts=%d", what, r->num_groups, r->num_experts);
    DPEP_REQUIRE(r->num_topk_groups >= 1 && r->num_topk_groups <= r->num_groups, "%s: num_topk_groups=%d is not in [1, num_groups]", what, r->num_topk_groups);
    DPEP_REQUIRE(r->num_topk <= r->num_topk_groups * (r->num_experts / r->num_groups), "%s: the chosen groups hold fewer than num_topk=%d experts", what, r->num_topk);
    DPEP_REQUIRE(r->score == DPEP_SCORE_SOFTMAX || r->score == DPEP_SCORE_SIGMOID, "%s: score=%d", what, r->score);
    DPEP_REQUIRE(r->logits_type >= DPEP_TYPE_F32 && r->logits_type <= DPEP_TYPE_F16, "%s: logits_type=%d", what, r->logits_type);
    DPEP_REQUIRE(r->index_bytes == 4 || r->index_bytes == 8, "%s: index_bytes=%d", what, r->index_bytes);
    DPEP_REQUIRE(r->scale == r->scale && r->scale != 0.0f && r->scale - r->scale == 0.0f, "%s: scale must be finite and not zero", what);
    return DPEP_OK;
}

}  // namespace
}  // namespace dpep

using namespace dpep;

extern "C" {

int dpep_route(const dpep_router* r, const void* logits, const float* bias, const uint8_t* token_mask, int num_tokens, void* topk_idx,
               float* topk_weights, void* stream)
{
    if (int rc = check_router(r, num_tokens, "route"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(bias == nullptr || r->score == DPEP_SCORE_SIGMOID, "route: a bias needs sigmoid scores");
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(logits != nullptr && topk_idx != nullptr && topk_weights != nullptr, "route: a NULL buffer");
    const Route call = {logits, bias, token_mask, topk_idx, topk_weights, num_tokens, r->num_experts, r->num_topk, r->num_groups, r->num_topk_groups,
                        r->normalize != 0, r->index_bytes == 8, r->scale};
    with_variant(r, [&](auto v, auto type, auto sigmoid) {
        route_kernel<v(), type(), sigmoid()><<<(num_tokens + kRouterWaves - 1) / kRouterWaves, kRouterThreads, 0, static_cast<hipStream_t>(stream)>>>(call);
    });
    return launch_status("route");
}

size_t dpep_balance_scratch_bytes(int num_experts, int num_tokens, int num_sequences)
{
    if (num_experts < 1 || num_tokens < 0 || num_sequences < 1) return 0;
    const size_t chunk = balance_chunk(num_tokens), rows = (num_tokens + chunk - 1) / chunk + num_sequences;
    return rows * (static_cast<size_t>(num_experts) * 8 + 4);
}

int dpep_balance_loss(const dpep_router* r, const void* logits, const void* topk_idx, int num_tokens, const int32_t* sequence_offsets, int num_sequences,
                      float* losses, int32_t* counts, int32_t* tokens, void* scratch, void* stream)
{
    if (int rc = check_router(r, num_tokens, "balance_loss"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(num_sequences >= 1 && (sequence_offsets != nullptr || num_sequences == 1), "balance_loss: num_sequences=%d", num_sequences);
    DPEP_REQUIRE(losses != nullptr && counts != nullptr && tokens != nullptr && scratch != nullptr, "balance_loss: a NULL buffer");
    DPEP_REQUIRE(num_tokens == 0 || (logits != nullptr && topk_idx != nullptr), "balance_loss: a NULL buffer");
    const int chunk = balance_chunk(num_tokens), chunks = (num_tokens + chunk - 1) / chunk;
    const size_t rows = static_cast<size_t>(chunks) + num_sequences;
    float* sums = static_cast<float*>(scratch);
    int32_t* partial_counts = reinterpret_cast<int32_t*>(sums + rows * r->num_experts);
    const Balance call = {logits, topk_idx, sequence_offsets, num_tokens, r->num_experts, r->num_topk, num_sequences, chunk, chunks, r->index_bytes == 8,
                          sums, partial_counts, partial_counts + rows * r->num_experts};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (chunks > 0)
        with_variant(r, [&](auto v, auto type, auto sigmoid) { balance_sums_kernel<v(), type(), sigmoid()><<<chunks, kRouterThreads, 0, s>>>(call); });
    balance_finish_kernel<<<num_sequences, kFinishThreads, 0, s>>>(call, losses, counts, tokens);
    return launch_status("balance_loss");
}

int dpep_router_backward(const dpep_router* r, const dpep_router_gradients* g, int num_tokens, void* stream)
{
    if (int rc = check_router(r, num_tokens, "router_backward"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(g != nullptr, "router_backward: gradients is NULL");
    DPEP_REQUIRE(g->grad_weights != nullptr || g->grad_losses != nullptr, "router_backward: neither grad_weights nor grad_losses is given");
    DPEP_REQUIRE(g->grad_losses == nullptr || (g->counts != nullptr && g->tokens != nullptr && g->num_sequences >= 1 &&
                                               (g->sequence_offsets != nullptr || g->num_sequences == 1)),
                 "router_backward: grad_losses needs the counts and tokens of its sequences");
    DPEP_REQUIRE(g->grad_weights == nullptr || !r->normalize || g->topk_weights != nullptr || num_tokens == 0, "router_backward: normalised weights are needed");
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(g->logits != nullptr && g->topk_idx != nullptr && g->grad_logits != nullptr, "router_backward: a NULL buffer");
    const bool balance = g->grad_losses != nullptr;
    const Backward call = {g->logits, g->topk_idx, g->topk_weights, g->grad_weights, g->sequence_offsets, balance ? g->counts : nullptr, g->tokens, g->grad_losses,
                           g->grad_logits, num_tokens, r->num_experts, r->num_topk, balance ? g->num_sequences : 1, r->normalize != 0, r->index_bytes == 8, r->scale};
    with_variant(r, [&](auto v, auto type, auto sigmoid) {
        router_backward_kernel<v(), type(), sigmoid()><<<(num_tokens + kRouterWaves - 1) / kRouterWaves, kRouterThreads, 0, static_cast<hipStream_t>(stream)>>>(call);
    });
    return launch_status("router_backward");
}

}  // extern "C"
