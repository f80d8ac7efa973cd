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
constexpr int kRouterThreads = 512;
constexpr int kRouterWaves = kRouterThreads / kWave;
constexpr int kMaxRouterExperts = 1024;
constexpr int kNone = INT32_MIN + 0x7fffff;  // the key of -inf: what is out of service ranks nowhere

// ---- a row in a wave's registers ---------------------------------------------------------------------------------------------------
template <int kControl>
__device__ __forceinline__ int dpp_or(int other, int v)
{
    return __builtin_amdgcn_update_dpp(other, v, kControl, 0xf, 0xf, false);
}
// Largest / sum over the wave, the same in every lane, by row shifts and row broadcasts (an LDS permute a step costs 50 ns and more).  Only lane 63 is
// looked at, so broadcasts go to all rows, which makes each step one instruction.
__device__ __forceinline__ int wave_max(int v)
{
    v = max(v, dpp_or<0x111>(INT32_MIN, v));  // row_shr:1
    v = max(v, dpp_or<0x112>(INT32_MIN, v));
    v = max(v, dpp_or<0x114>(INT32_MIN, v));
    v = max(v, dpp_or<0x118>(INT32_MIN, v));
    v = max(v, dpp_or<0x142>(INT32_MIN, v));  // row_bcast:15
    v = max(v, dpp_or<0x143>(INT32_MIN, v));  // row_bcast:31
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ float wave_sum(float v)
{
    auto add = [&](int shifted) { v += __int_as_float(shifted); };
    add(dpp_or<0x111>(0, __float_as_int(v)));
    add(dpp_or<0x112>(0, __float_as_int(v)));
    add(dpp_or<0x114>(0, __float_as_int(v)));
    add(dpp_or<0x118>(0, __float_as_int(v)));
    add(dpp_or<0x142>(0, __float_as_int(v)));
    add(dpp_or<0x143>(0, __float_as_int(v)));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Integers in the order of the floats (no NaN and no -0: adding +0, or a sum of a score and anything, leaves none).
__device__ __forceinline__ int ordered(float v)
{
    const int bits = __float_as_int(v);
    return bits ^ static_cast<int>(static_cast<uint32_t>(bits >> 31) >> 1);
}
__device__ __forceinline__ float unordered(int key) { return __int_as_float(key ^ ((key >> 31) & 0x7fffffff)); }

// What the wave's lanes stored to LDS is there for all of them.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int kType>
using Logit = std::conditional_t<kType == DPEP_TYPE_F32, uint32_t, uint16_t>;
template <int kType>
__device__ __forceinline__ float widen(uint32_t bits)
{
    if constexpr (kType == DPEP_TYPE_F32) return __uint_as_float(bits);
    if constexpr (kType == DPEP_TYPE_BF16) return bf16_to_f32(bits);
    return f16_to_f32(bits);
}
template <int kType>
__device__ __forceinline__ float load_logit(const void* p, size_t i)
{
    return widen<kType>(static_cast<const Logit<kType>*>(p)[i]);
}
// V values next to one another as the memory holds them: in one piece where rows allow it (whole: the number of experts is a multiple of V and rows
// are aligned to pieces), else one by one.
template <int V, int kType>
struct Piece {
    using Word = Logit<kType>;
    static constexpr int kBytes = V * sizeof(Word);
    using Part = std::conditional_t<kBytes >= 16, u32x4, std::conditional_t<kBytes == 8, u32x2, std::conditional_t<kBytes == 4, uint32_t, Word>>>;
    static constexpr int kParts = kBytes / sizeof(Part);
    Word at[V];
    __device__ __forceinline__ void load(const void* rows, size_t row, int experts, int lane, bool whole)
    {
        const Word* const from = static_cast<const Word*>(rows) + row;
        const int first = lane * V;
        if (whole) {
            const int clamped = first < experts ? first : 0;
            const Part* const parts = reinterpret_cast<const Part*>(from + clamped);
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const Part part = parts[i];
                __builtin_memcpy(at + i * (V / kParts), &part, sizeof(Part));
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) at[v] = from[min(first + v, experts - 1)];
        }
    }
    __device__ __forceinline__ void store(void* rows, size_t row, int experts, int lane, bool whole) const
    {
        Word* const to = static_cast<Word*>(rows) + row;
        const int first = lane * V;
        if (whole) {
            if (first < experts)
#pragma unroll
                for (int i = 0; i < kParts; ++i) {
                    Part part;
                    __builtin_memcpy(&part, at + i * (V / kParts), sizeof(Part));
                    reinterpret_cast<Part*>(to + first)[i] = part;
                }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (first + v < experts) to[first + v] = at[v];
        }
    }
    __device__ __forceinline__ float value(int v, int experts, int lane) const { return lane * V + v < experts ? widen<kType>(at[v]) : -kInf; }
    __device__ __forceinline__ void set(int v, float value)
    {
        if constexpr (kType == DPEP_TYPE_F32) at[v] = __float_as_uint(value);
        if constexpr (kType == DPEP_TYPE_BF16) at[v] = static_cast<uint16_t>(f32_to_bf16(value));
        if constexpr (kType == DPEP_TYPE_F16) at[v] = static_cast<uint16_t>(pack_f16x2(value, 0.0f) & 0xffffu);
    }
};
// Id of a slot of the row that begins at id `row` (the same in all lanes).
__device__ __forceinline__ int load_index(const void* p, bool wide, size_t row, int slot, int experts)
{
    const long long e = wide ? (static_cast<const int64_t*>(p) + row)[slot] : (static_cast<const int32_t*>(p) + row)[slot];
    return e >= 0 && e < experts ? static_cast<int>(e) : -1;
}

// 1 / (1 + exp(-z)) as IEEE divide and the library's exp give it, bit for bit (the choice compares such values, so everybody has to get the
// same): one step from the hardware's reciprocal is correctly rounded for every mantissa and exponent below 2^126 (the tests compare
// every float's), and beyond that, below a logit of -86, the divide itself is taken.  grown: exp(-z).
__device__ __forceinline__ float sigmoid_of(float grown)
{
    const float d = 1.0f + grown, r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.0f), r, r);
}
template <int V>
__device__ __forceinline__ void sigmoids(const float (&z)[V], float (&s)[V], float (&grown)[V])
{
    unsigned long long far = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        grown[v] = expf(-z[v]);
        s[v] = sigmoid_of(grown[v]);
        far |= __ballot(z[v] < -86.0f) & ~__ballot(z[v] == -kInf);
    }
    if (far != 0)
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = 1.0f / (1.0f + grown[v]);
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (z[v] == -kInf) s[v] = 0.0f;
}
__device__ __forceinline__ float sigmoid(float z)
{
    const float z1[1] = {z};
    float s[1], grown[1];
    sigmoids<1>(z1, s, grown);
    return s[0];
}
__device__ __forceinline__ float reciprocal(float d)  // of 1e-20 .. 1e30
{
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.0f), r, r);
}

// A row's scores: exp(z - max) or the sigmoids, and 1 / their sum (the balance loss's probabilities are their products).  grown: exp(-z) (sigmoid).
template <int V, bool kSigmoid>
__device__ __forceinline__ float row_scores(const float (&z)[V], float (&s)[V], float (&grown)[V])
{
    float total = 0.0f;
    if constexpr (kSigmoid) {
        sigmoids<V>(z, s, grown);
    } else {
        int top = kNone;
#pragma unroll
        for (int v = 0; v < V; ++v) top = max(top, ordered(z[v] == z[v] ? z[v] : -kInf));
        const float largest = unordered(wave_max(top));
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = z[v] == -kInf ? 0.0f : expf(z[v] - largest);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) total += s[v];
    total = wave_sum(total);
    return kSigmoid ? reciprocal(total + kTiny) : total == 0.0f ? 0.0f : 1.0f / total;
}

// ---- sequences -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int sequence_begin(const int32_t* offsets, int b, int sequences, int tokens)
{
    if (b >= sequences) return tokens;
    if (offsets == nullptr) return b == 0 ? 0 : tokens;
    return min(max(offsets[b], 0), tokens);
}
// The last sequence that begins at `token` (the same in all lanes) or in front of it: 64 are looked at in a step.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int sequences, int token, int lane)
{
    if (offsets == nullptr) return 0;
    int low = 0, high = sequences;
    while (high - low > 1) {
        const int step = (high - low + kWave - 1) / kWave, at = low + lane * step;
        const int begun = __popcll(__ballot(at < high && offsets[min(at, high - 1)] <= token));
        low += max(begun - 1, 0) * step;
        high = min(low + step, high);
    }
    return low;
}

// ---- choice and balance sums --------------------------------------------------------------------------------------------------------
struct Forward {
    const void* logits;
    // choice
    const float* bias;
    const uint8_t* token_mask;
    void* topk_idx;
    float* topk_weights;
    int groups, topk_groups;
    int group_lanes;  // a group's lanes where groups are 1, 2, 4 .. 16 lanes of whole registers, else 0
    bool normalize;
    float scale;
    // sums of the balance loss.  Chunks of tokens (a workgroup each) leave one row of sums for every sequence that they touch; (chunk + sequence)
    // numbers these rows.
    const int32_t* offsets;
    int sequences;
    float* sums;       // [chunks + sequences][experts]: of the probabilities
    int32_t* counts;   // the same: routes
    int32_t* members;  // [chunks + sequences]: tokens with a route
    uint32_t* tickets; // [sequences]
    int tokens, experts, topk, chunk;
    bool wide, whole;
};

// Keys of experts outside the best groups become kNone.  Groups of whole lanes: a lane's two largest, then the group's by exchanges among its lanes;
// other groups one after the other, each over the whole wave.  A group's rank is how many are ahead of it.
template <int V, bool kSigmoid>
__device__ __forceinline__ void limit_groups(int (&key)[V], const Forward& c, int lane)
{
    auto score = [](int first, int second) {
        return !kSigmoid || second == kNone ? first : ordered(fminf(unordered(first) + unordered(second), kInf));
    };
    auto two_largest = [&](const int (&of)[V], int& first, int& second) {
        first = of[0];
        second = kNone;
#pragma unroll
        for (int v = 1; v < V; ++v) {
            second = max(second, min(first, of[v]));
            first = max(first, of[v]);
        }
    };
    // lane g * stride (a group's first lane, or lane g) has group g's score
    auto ahead_of = [&](int mine, int stride) {
        int ahead = 0;
        for (int o = 0; o < c.groups; ++o) {
            const int other = __builtin_amdgcn_readlane(mine, o * stride), behind = (o + 1) * stride;  // (lanes of later groups lose a tie)
            const unsigned long long later = behind < kWave ? ~0ull << behind : 0ull;
            ahead += __builtin_amdgcn_inverse_ballot_w64(__ballot(other > mine) | (__ballot(other == mine) & later));
        }
        return ahead;
    };
    if (c.group_lanes > 0) {
        int first, second;
        two_largest(key, first, second);
        auto merge = [&](auto control) {
            const int other = dpp_or<control()>(kNone, first), other_second = dpp_or<control()>(kNone, second);
            second = max(max(second, other_second), min(first, other));
            first = max(first, other);
        };
        if (c.group_lanes >= 2) merge(std::integral_constant<int, 0xB1>{});    // lane ^ 1
        if (c.group_lanes >= 4) merge(std::integral_constant<int, 0x4E>{});    // lane ^ 2
        if (c.group_lanes >= 8) merge(std::integral_constant<int, 0x141>{});   // the other four of eight
        if (c.group_lanes >= 16) merge(std::integral_constant<int, 0x140>{});  // the other eight of sixteen
        const int mine = score(first, second);
        int ahead;
        if (c.groups <= c.group_lanes) {
            // a group's lane j compares it with group j: its share of the ballot is who is ahead
            const int other = __builtin_amdgcn_ds_bpermute((lane & (c.group_lanes - 1)) * c.group_lanes * 4, mine);
            const int group_first = lane & -c.group_lanes, j = lane - group_first;
            const bool is_ahead = j < c.groups && (other > mine || (other == mine && j * c.group_lanes < group_first));
            ahead = __popc(static_cast<uint32_t>(__ballot(is_ahead) >> group_first) & ((1u << c.group_lanes) - 1));
        } else {
            ahead = ahead_of(mine, c.group_lanes);
        }
        const bool out = ahead >= c.topk_groups;
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = out ? kNone : key[v];
        return;
    }
    const int width = c.experts / c.groups;
    int mine = kNone;
    for (int g = 0; g < c.groups; ++g) {
        int in[V], first, second;
#pragma unroll
        for (int v = 0; v < V; ++v) in[v] = static_cast<unsigned>(lane * V + v - g * width) < static_cast<unsigned>(width) ? key[v] : kNone;
        two_largest(in, first, second);
        const int largest = wave_max(first), owner = __ffsll(__ballot(first == largest)) - 1;
        const int of_group = score(largest, wave_max(lane == owner ? second : first));
        mine = lane == g ? of_group : mine;
    }
    const unsigned long long out = __ballot(ahead_of(mine, 1) >= c.topk_groups);
    for (int g = 0; g < c.groups; ++g)
        if ((out >> g) & 1)
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = static_cast<unsigned>(lane * V + v - g * width) < static_cast<unsigned>(width) ? kNone : key[v];
}

// Sorts a lane's keys, largest first and equal ones in their order (neighbours change places only where the second is larger), and packs where they
// were, a byte each (V == 16: half a byte).
template <int V>
struct Places {
    static constexpr int kBits = V == 16 ? 4 : 8;
    using Word = std::conditional_t<V <= 4, uint32_t, uint64_t>;
    Word word;
};
template <int V>
__device__ __forceinline__ Places<V> sort_keys(int (&key)[V])
{
    int at[V];
#pragma unroll
    for (int v = 0; v < V; ++v) at[v] = v;
#pragma unroll
    for (int turn = 0; turn < V; ++turn)
#pragma unroll
        for (int a = turn & 1; a + 1 < V; a += 2) {
            // (by value: a choice between elements would become one between their addresses)
            const int x = key[a], y = key[a + 1], at_x = at[a], at_y = at[a + 1];
            key[a] = max(x, y);
            key[a + 1] = min(x, y);
            at[a] = y > x ? at_y : at_x;
            at[a + 1] = y > x ? at_x : at_y;
        }
    Places<V> places = {0};
#pragma unroll
    for (int v = 0; v < V; ++v) places.word |= static_cast<typename Places<V>::Word>(at[v]) << (Places<V>::kBits * v);
    return places;
}

// Lane k gets the expert of slot k, -1 where none is left: each time the largest key of the wave, in its lowest lane (experts are counted along lanes,
// and a lane's equal keys stand in their order, so that is the lowest index).  Every lane's keys are sorted first: a step then compares and
// removes heads alone.  (Finding the register of the largest key in each step takes 45 scalar instructions, which issue no faster than the
// 17 of the vector unit beside them.)
template <int V>
__device__ __forceinline__ int choose(int (&left)[V], int topk)
{
    int mine = -1;
    Places<V> places = sort_keys(left);
    for (int k = 0; k < topk; ++k) {
        const int largest = wave_max(left[0]);
        if (largest == kNone) break;
        const int lane = __builtin_ctzll(__ballot(left[0] == largest));
        const int expert = lane * V + (__builtin_amdgcn_readlane(static_cast<int>(places.word), lane) & ((1 << Places<V>::kBits) - 1));
        mine = __builtin_amdgcn_inverse_ballot_w64(1ull << k) ? expert : mine;
        const bool taken = __builtin_amdgcn_inverse_ballot_w64(1ull << lane);
#pragma unroll
        for (int v = 0; v < V; ++v) left[v] = !taken ? left[v] : v + 1 < V ? left[v + 1] : kNone;
        places.word = taken ? places.word >> Places<V>::kBits : places.word;
    }
    return mine;
}

// In lane k: the value that belongs to expert `mine` (0 where there is none) of a row in the wave's registers.
template <int V>
__device__ __forceinline__ float pick(const float (&x)[V], int mine)
{
    const int owner = max(mine, 0) / V;
    float found = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float other = __int_as_float(__builtin_amdgcn_ds_bpermute(owner * 4, __float_as_int(x[v])));
        found = mine == owner * V + v ? other : found;
    }
    return found;
}

// A wave takes every eighth token of a workgroup's chunk, the whole row in its registers, so logits are read once and the choice, the weights and the
// balance sums come out of one pass.  Vector instructions bound it, not HBM: 65536 x 256 in eight groups, sigmoid, K = 8, with the sums takes
// 57 us (409 vector instructions a token, 43 us of issue; its 72 MB take 14), 128 x 384 4.8, one token 3.4.  Half of the instructions are the
// exponentials and the eight steps of the choice.  Rows of more than 512 experts take sixteen registers a lane for each of their arrays: of those, 15 go to
// the stack in a sigmoid route of FP32 logits, 28 to 36 where balance sums are taken with the choice.
template <int V, int kType, bool kSigmoid, bool kRoute, bool kBalance>
__global__ __launch_bounds__(kRouterThreads) void router_forward_kernel(const Forward c)
{
    __shared__ float rows_lds[kBalance ? kRouterWaves : 1][kWave * V];  // the waves' sums
    __shared__ int counts[kBalance ? kWave * V : 1];
    __shared__ int members[kRouterWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = blockIdx.x * c.chunk, last = min(first + c.chunk, c.tokens);
    if (kBalance && blockIdx.x == 0)
        for (int b = threadIdx.x; b < c.sequences; b += kRouterThreads) c.tickets[b] = 0;
    float bias[V];
    if constexpr (kRoute && kSigmoid)
#pragma unroll
        for (int v = 0; v < V; ++v) bias[v] = c.bias != nullptr && lane * V + v < c.experts ? c.bias[lane * V + v] : 0.0f;

    int begin = first;
    for (int b = kBalance ? sequence_of(c.offsets, c.sequences, first, lane) : 0; begin < last && b < c.sequences; ++b) {
        const int end = !kBalance || b + 1 == c.sequences ? last : min(last, sequence_begin(c.offsets, b + 1, c.sequences, c.tokens));
        if (end <= begin) continue;
        float sum[V] = {};
        int held = 0;
        if constexpr (kBalance) {
            for (int e = threadIdx.x; e < c.experts; e += kRouterThreads) counts[e] = 0;
            __syncthreads();
        }
        // (what the next token needs is asked for while this one is worked on)
        Piece<V, kType> next;
        int next_route = -1;
        uint8_t next_real = 1;
        auto fetch = [&](int t) {
            if (t >= end) return;
            next.load(c.logits, static_cast<size_t>(t) * c.experts, c.experts, lane, c.whole);
            if constexpr (kRoute) next_real = c.token_mask == nullptr ? 1 : c.token_mask[t];
            else next_route = lane < c.topk ? load_index(c.topk_idx, c.wide, static_cast<size_t>(t) * c.topk, lane, c.experts) : -1;
        };
        fetch(begin + wave);
        for (int t = begin + wave; t < end; t += kRouterWaves) {
            const size_t to = static_cast<size_t>(t) * c.topk;
            const Piece<V, kType> piece = next;
            const bool real = __builtin_amdgcn_readfirstlane(next_real) != 0;
            int mine = kRoute ? -1 : next_route;
            fetch(t + kRouterWaves);
            float z[V], s[V], grown[V], inverse = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) z[v] = piece.value(v, c.experts, lane);
            if (kBalance || (!kSigmoid && !c.normalize)) inverse = row_scores<V, kSigmoid>(z, s, grown);
            else if constexpr (kSigmoid) sigmoids<V>(z, s, grown);
            if constexpr (kRoute) {
                if (real) {
                    int key[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        // a NaN ranks with +inf, so that it is chosen and shows in the weights
                        const float k = !kSigmoid ? z[v] + 0.0f : z[v] == -kInf ? -kInf : s[v] + bias[v];
                        key[v] = ordered(fminf(k, kInf));
                    }
                    if (c.groups > 1) limit_groups<V, kSigmoid>(key, c, lane);
                    mine = choose<V>(key, c.topk);
                }
                float weight;
                if constexpr (kSigmoid) {
                    weight = pick<V>(s, mine);
                    if (c.normalize) weight = weight / (wave_sum(weight) + kTiny);
                } else if (c.normalize) {
                    const float picked = pick<V>(z, mine), chosen = mine >= 0 ? picked : -kInf;
                    const float top = unordered(wave_max(chosen == chosen ? ordered(chosen) : kNone));
                    weight = mine >= 0 ? expf(chosen - top) : 0.0f;
                    const float total = wave_sum(weight);
                    weight = mine >= 0 ? weight / total : 0.0f;
                } else {
                    weight = pick<V>(s, mine) * inverse;
                }
                if (lane < c.topk) {
                    if (c.wide) (static_cast<int64_t*>(c.topk_idx) + to)[lane] = mine;
                    else (static_cast<int32_t*>(c.topk_idx) + to)[lane] = mine;
                    // (not a product: a slot without an expert weighs 0 whatever the row holds, and padding rows may hold anything)
                    (c.topk_weights + to)[lane] = mine >= 0 ? weight * c.scale : 0.0f;
                }
            }
            if constexpr (kBalance) {
                if (__ballot(mine >= 0) == 0) continue;
                if (mine >= 0) atomicAdd(&counts[mine], 1);
                ++held;
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] = fmaf(s[v], inverse, sum[v]);
            }
        }
        if constexpr (kBalance) {
            wave_sync();
#pragma unroll
            for (int v = 0; v < V; ++v) rows_lds[wave][lane * V + v] = sum[v];
            if (lane == 0) members[wave] = held;
            __syncthreads();
            const size_t slot = blockIdx.x + b;
            for (int e = threadIdx.x; e < c.experts; e += kRouterThreads) {
                float total = 0.0f;
#pragma unroll
                for (int w = 0; w < kRouterWaves; ++w) total += rows_lds[w][e];
                c.sums[slot * c.experts + e] = total;
                c.counts[slot * c.experts + e] = counts[e];
            }
            if (threadIdx.x == 0) {
                int total = 0;
                for (int w = 0; w < kRouterWaves; ++w) total += members[w];
                c.members[slot] = total;
            }
            __syncthreads();
        }
        begin = end;
    }
}

// Sequence b of N tokens with a route and R routes, c_e of them to expert e; p a token's softmax, or its sigmoids over their sum:
//   f_e = E c_e / R,  loss_b = sum_e f_e (sum_t p_te) / N = E / (R N) sum_e c_e sum_t p_te
// A workgroup adds up 64 experts' rows of sums, sixteen at a time; the last of a sequence's workgroups has the loss.  (A few dependent trips to
// memory: 6.0 us for 1024 rows of 256 experts in 16 sequences, 3.2 for the 25 of 777 tokens.)
constexpr int kFinishWaves = 16;
struct Finish {
    const float* sums;
    const int32_t* counts;
    const int32_t* members;
    const int32_t* offsets;
    uint32_t* tickets;
    float* products;  // [sequences][pieces of 64 experts]
    int32_t* routes;  // the same
    float* losses;
    int32_t* all_counts;
    int32_t* all_members;
    int tokens, experts, sequences, chunk;
};
__global__ __launch_bounds__(kFinishWaves * kWave) void balance_finish_kernel(const Finish c)
{
    __shared__ float part[kFinishWaves][kWave];
    __shared__ int part_count[kFinishWaves][kWave];
    __shared__ int part_members[kFinishWaves];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.y * kWave + lane;
    const int begin = sequence_begin(c.offsets, b, c.sequences, c.tokens), end = sequence_begin(c.offsets, b + 1, c.sequences, c.tokens);
    const int first = begin / c.chunk, last = end > begin ? (end - 1) / c.chunk : first - 1;
    float sum = 0.0f;
    int count = 0, held = 0;
    const int at = min(e, c.experts - 1);
#pragma unroll 4
    for (int i = first + wave; i <= last; i += kFinishWaves) {
        const size_t row = static_cast<size_t>(i + b);
        sum += c.sums[row * c.experts + at];
        count += c.counts[row * c.experts + at];
        held += c.members[row];
    }
    part[wave][lane] = sum;
    part_count[wave][lane] = count;
    if (lane == 0) part_members[wave] = held;
    __syncthreads();
    if (wave != 0) return;
    sum = 0.0f;
    count = held = 0;
#pragma unroll
    for (int w = 0; w < kFinishWaves; ++w) {
        sum += part[w][lane];
        count += part_count[w][lane];
        held += part_members[w];
    }
    if (e < c.experts) c.all_counts[static_cast<size_t>(b) * c.experts + e] = count;
    else count = 0;
    const float product = wave_sum(sum * static_cast<float>(count));
    const int routes = wave_total(count);
    if (lane != 0) return;
    // (relaxed stores that go past this die's cache, then the ticket; the last one reads them the same way)
    const int pieces = gridDim.y;
    __hip_atomic_store(c.products + b * pieces + blockIdx.y, product, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(c.routes + b * pieces + blockIdx.y, routes, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t ticket = __hip_atomic_fetch_add(c.tickets + b, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    if (ticket != static_cast<uint32_t>(pieces) - 1) return;
    float all = 0.0f;
    int total = 0;
    for (int i = 0; i < pieces; ++i) {
        all += __hip_atomic_load(c.products + b * pieces + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        total += __hip_atomic_load(c.routes + b * pieces + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    c.losses[b] = held > 0 ? all / static_cast<float>(held) * (static_cast<float>(c.experts) / static_cast<float>(total)) : 0.0f;
    c.all_members[b] = held;
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
    int tokens, experts, topk, sequences, chunk;
    bool normalize, wide, whole;
    float scale, inverse_scale;
};

// With w a token's weights over the scale, g their gradients times the scale, p the scores, a = the loss's gradient over the sequence's N, f its loads:
//   softmax, normalised  w_k (g_k - sum g w) at the chosen;  not normalised  p_e ([e chosen] g_e - sum g p)
//   sigmoid  g'_k s_k (1 - s_k) at the chosen, g' = g, or normalised (g_k - sum g w) / (sum s + 1e-20)
//   balance  softmax a p_e (f_e - sum f p);  sigmoid a (f_e - sum f p) s_e (1 - s_e) / (sum s + 1e-20)
// A wave takes a token: what belongs to the chosen is scattered into its row in LDS, so the row leaves once, in whole lines.  Scores are taken
// again from the logits, which costs less than to keep them (a row of FP32 written and read).  65536 x 256 with both gradients: 41 us = 3.4 TB/s of
// logits and gradient (25 us of it vector issue); 4096 x 128 with the weights' alone, which reads no row: 3.4 us.
template <int V, int kType, bool kSigmoid>
__global__ __launch_bounds__(kRouterThreads) void router_backward_kernel(const Backward c)
{
    __shared__ __attribute__((aligned(16))) float rows[kRouterWaves][kWave * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = blockIdx.x * c.chunk, last = min(first + c.chunk, c.tokens);
    const bool dense = c.grad_weights != nullptr && !kSigmoid && !c.normalize, balance = c.counts != nullptr;
    float* const mine = rows[wave];
    // the sequence of the token at hand: its loads f, where it ends, and grad / N
    float f[V] = {}, of_loss = 0.0f;
    int sequence = -1, sequence_end = 0;
    Piece<V, kType> next = {};
    int next_route = -1;
    float next_grad = 0.0f, next_weight = 0.0f;
    auto fetch = [&](int t) {
        if (t >= last) return;
        const size_t slots = static_cast<size_t>(t) * c.topk;
        if (dense || balance) next.load(c.logits, static_cast<size_t>(t) * c.experts, c.experts, lane, c.whole);
        if (lane >= c.topk) return;
        next_route = load_index(c.topk_idx, c.wide, slots, lane, c.experts);
        if (c.grad_weights != nullptr) {
            next_grad = (c.grad_weights + slots)[lane];
            if (c.normalize) next_weight = (c.topk_weights + slots)[lane];
        }
    };
    fetch(first + wave);
    for (int t = first + wave; t < last; t += kRouterWaves) {
        const size_t row = static_cast<size_t>(t) * c.experts;
        const Piece<V, kType> piece = next;
        const int e = next_route;
        const float through_weight = next_grad, weight_of_route = next_weight;
        fetch(t + kRouterWaves);
        const bool padding = __ballot(e >= 0) == 0;
        float grad[V] = {}, s[V] = {}, grown[V] = {}, inverse = 0.0f;
        if (!padding && (dense || balance)) {
            float z[V];
#pragma unroll
            for (int v = 0; v < V; ++v) z[v] = piece.value(v, c.experts, lane);
            inverse = row_scores<V, kSigmoid>(z, s, grown);
            if (balance) {
                // softmax: a p (f - sum f p); sigmoid: a s (1 - s) / sum s (f - sum f p);  a = grad / N
                if (t >= sequence_end) {
                    sequence = sequence < 0 ? sequence_of(c.offsets, c.sequences, t, lane) : sequence;
                    while (sequence + 1 < c.sequences && sequence_begin(c.offsets, sequence + 1, c.sequences, c.tokens) <= t) ++sequence;
                    sequence_end = sequence_begin(c.offsets, sequence + 1, c.sequences, c.tokens);
                    int routes = 0;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const int at = lane * V + v, count = at < c.experts ? c.counts[static_cast<size_t>(sequence) * c.experts + at] : 0;
                        routes += count;
                        f[v] = static_cast<float>(count);
                    }
                    routes = wave_total(routes);
                    const float unit = routes > 0 ? static_cast<float>(c.experts) / static_cast<float>(routes) : 0.0f;
#pragma unroll
                    for (int v = 0; v < V; ++v) f[v] *= unit;
                    of_loss = c.grad_losses[sequence] / static_cast<float>(max(c.members[sequence], 1));
                }
                float mean = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) mean += f[v] * (s[v] * inverse);
                mean = wave_sum(mean);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    // 1 - s = exp(-z) s (the difference would cancel); where exp(-z) is past the range, s is 0
                    const float slope = kSigmoid ? s[v] * (fminf(grown[v], 3e38f) * s[v]) : s[v];
                    grad[v] = of_loss * (f[v] - mean) * (z[v] == -kInf ? 0.0f : slope * inverse);
                }
            }
        }
        if (c.grad_weights != nullptr && !padding) {
#pragma unroll
            for (int v = 0; v < V; ++v) mine[lane * V + v] = 0.0f;
            wave_sync();
            float g = e >= 0 ? through_weight * c.scale : 0.0f, through = 0.0f;
            if (c.normalize) {
                const float w = e >= 0 ? weight_of_route * c.inverse_scale : 0.0f;
                const float inner = wave_sum(g * w);
                g = e >= 0 ? g - inner : 0.0f;
                through = w * g;
            }
            if constexpr (kSigmoid) {
                float score, of_exp;
                if (balance) {
                    score = pick<V>(s, e);
                    of_exp = pick<V>(grown, e);
                } else {
                    const float z = e >= 0 ? load_logit<kType>(c.logits, row + e) : 0.0f;
                    of_exp = expf(-z);
                    score = e >= 0 ? sigmoid(z) : 0.0f;
                }
                through = g * score * (fminf(of_exp, 3e38f) * score);
                if (c.normalize) through = through * reciprocal(wave_sum(score) + kTiny);
            }
            if (e >= 0) atomicAdd(&mine[e], dense ? g : through);
            wave_sync();
            float own[V];
#pragma unroll
            for (int v = 0; v < V; ++v) own[v] = mine[lane * V + v];
            if (dense) {
                // p_e ([e chosen] g_e - sum_j g_j p_j)
                float inner = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) inner += own[v] * (s[v] * inverse);
                inner = wave_sum(inner);
#pragma unroll
                for (int v = 0; v < V; ++v) grad[v] += s[v] * inverse * (own[v] - inner);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) grad[v] += own[v];
            }
            wave_sync();
        }
        Piece<V, kType> out;
#pragma unroll
        for (int v = 0; v < V; ++v) out.set(v, grad[v]);
        out.store(c.grad_logits, row, c.experts, lane, c.whole);
    }
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

// Registers of a lane for a number of experts, as with_variant chooses them.
int row_registers(int experts)
{
    int v = 1;
    while (v * kWave < experts) v *= 2;
    return v;
}
// Whether rows of `experts` logits can be read in pieces of a lane's registers.
bool whole_pieces(const dpep_router* r, const void* a, const void* b)
{
    const size_t piece = std::min<size_t>(16, row_registers(r->num_experts) * (r->logits_type == DPEP_TYPE_F32 ? 4 : 2));
    return r->num_experts % row_registers(r->num_experts) == 0 && (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % piece == 0;
}
// Tokens to a workgroup: at most 1024 workgroups of eight waves, four to a CU where registers allow it (up to 128 experts; choice and sums
// together over 256 take up to 68 registers, three at once, and wider rows more); rows of sums stay few.
int router_chunk(int tokens) { return std::max(kRouterWaves, (tokens + 1023) / 1024); }
// With balance sums at least four tokens to a wave: a workgroup leaves a row of sums, which costs about as much as a token and is read again.
int balance_chunk(int tokens) { return std::max(4 * kRouterWaves, (tokens + 1023) / 1024); }

// Scratch of a balance loss.
struct BalanceScratch {
    size_t counts, members, tickets, products, routes, bytes;
    BalanceScratch(int experts, int tokens, int sequences)
    {
        const size_t chunk = balance_chunk(tokens), rows = (tokens + chunk - 1) / chunk + sequences, pieces = (experts + kWave - 1) / kWave;
        counts = rows * experts * 4;
        members = counts + rows * experts * 4;
        tickets = members + rows * 4;
        products = tickets + static_cast<size_t>(sequences) * 4;
        routes = products + sequences * pieces * 4;
        bytes = routes + sequences * pieces * 4;
    }
};

int check_router(const dpep_router* r, int num_tokens, const char* what)
{
    DPEP_REQUIRE(r != nullptr, "%s: router is NULL", what);
    DPEP_REQUIRE(num_tokens >= 0 && num_tokens <= DPEP_MAX_ROUTER_TOKENS, "%s: num_tokens=%d is not in [0, 2^30]", what, num_tokens);
    DPEP_REQUIRE(r->num_experts >= 1 && r->num_experts <= kMaxRouterExperts, "%s: num_experts=%d is not in [1, %d]", what, r->num_experts, kMaxRouterExperts);
    DPEP_REQUIRE(r->num_topk >= 1 && r->num_topk <= DPEP_MAX_TOPK && r->num_topk <= r->num_experts, "%s: num_topk=%d is not in [1, min(%d, num_experts)]", what,
                 r->num_topk, DPEP_MAX_TOPK);
    DPEP_REQUIRE(r->num_groups >= 1 && r->num_experts % r->num_groups == 0, "%s: num_groups=%d does not divide num_experts=%d", what, r->num_groups, r->num_experts);
    DPEP_REQUIRE(r->num_groups <= kWave, "%s: num_groups=%d is more than %d", what, r->num_groups, kWave);
    DPEP_REQUIRE(r->num_topk_groups >= 1 && r->num_topk_groups <= r->num_groups, "%s: num_topk_groups=%d is not in [1, num_groups]", what, r->num_topk_groups);
    DPEP_REQUIRE(r->num_topk <= r->num_topk_groups * (r->num_experts / r->num_groups), "%s: the chosen groups hold fewer than num_topk=%d experts", what, r->num_topk);
    DPEP_REQUIRE(r->score == DPEP_SCORE_SOFTMAX || r->score == DPEP_SCORE_SIGMOID, "%s: score=%d", what, r->score);
    DPEP_REQUIRE(r->logits_type >= DPEP_TYPE_F32 && r->logits_type <= DPEP_TYPE_F16, "%s: logits_type=%d", what, r->logits_type);
    DPEP_REQUIRE(r->index_bytes == 4 || r->index_bytes == 8, "%s: index_bytes=%d", what, r->index_bytes);
    DPEP_REQUIRE(r->scale >= 1e-30f && r->scale <= 1e30f || r->scale <= -1e-30f && r->scale >= -1e30f, "%s: scale must be of 1e-30 to 1e30 in magnitude", what);
    return DPEP_OK;
}

}  // namespace
}  // namespace dpep

using namespace dpep;

namespace {

// Choice (out: topk_idx, topk_weights), balance sums, or both in one pass.
int run_forward(const dpep_router* r, Forward call, int num_tokens, bool route, bool balance, float* losses, int32_t* counts, int32_t* tokens, void* scratch,
                void* stream, const char* what)
{
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int experts = r->num_experts, v = row_registers(experts), width = experts / r->num_groups;
    call.groups = r->num_groups;
    call.topk_groups = r->num_topk_groups;
    call.group_lanes = width % v == 0 && width / v <= 16 && (width / v & (width / v - 1)) == 0 ? width / v : 0;
    call.normalize = r->normalize != 0;
    call.scale = r->scale;
    call.tokens = num_tokens;
    call.experts = experts;
    call.topk = r->num_topk;
    call.chunk = balance ? balance_chunk(num_tokens) : router_chunk(num_tokens);
    call.wide = r->index_bytes == 8;
    call.whole = whole_pieces(r, call.logits, nullptr);
    const BalanceScratch at(experts, num_tokens, call.sequences);
    unsigned char* const base = static_cast<unsigned char*>(scratch);
    if (balance) {
        call.sums = reinterpret_cast<float*>(base);
        call.counts = reinterpret_cast<int32_t*>(base + at.counts);
        call.members = reinterpret_cast<int32_t*>(base + at.members);
        call.tickets = reinterpret_cast<uint32_t*>(base + at.tickets);
    }
    const int chunks = std::max(1, (num_tokens + call.chunk - 1) / call.chunk);  // (without tokens: the one that clears the tickets)
    with_variant(r, [&](auto registers, auto type, auto sigmoid) {
        if (route && balance) router_forward_kernel<registers(), type(), sigmoid(), true, true><<<chunks, kRouterThreads, 0, s>>>(call);
        else if (route) router_forward_kernel<registers(), type(), sigmoid(), true, false><<<chunks, kRouterThreads, 0, s>>>(call);
        else router_forward_kernel<registers(), type(), sigmoid(), false, true><<<chunks, kRouterThreads, 0, s>>>(call);
    });
    if (balance) {
        const Finish finish = {call.sums, call.counts, call.members, call.offsets, call.tickets, reinterpret_cast<float*>(base + at.products),
                               reinterpret_cast<int32_t*>(base + at.routes), losses, counts, tokens, num_tokens, experts, call.sequences, call.chunk};
        balance_finish_kernel<<<dim3(call.sequences, (experts + kWave - 1) / kWave), kFinishWaves * kWave, 0, s>>>(finish);
    }
    return launch_status(what);
}

// A sequence's routes are counted in 32 bits.
int check_routes(const dpep_router* r, int num_tokens, const char* what)
{
    DPEP_REQUIRE(static_cast<long long>(num_tokens) * r->num_topk < (1ll << 31), "%s: T*K must fit int32", what);
    return DPEP_OK;
}

int check_balance(const dpep_router* r, int num_tokens, const int32_t* sequence_offsets, int num_sequences, const float* losses, const int32_t* counts,
                  const int32_t* tokens, const void* scratch, const char* what)
{
    if (int rc = check_routes(r, num_tokens, what); rc != DPEP_OK) return rc;
    // (a workgroup of 1024 lanes to a sequence, and a launch's lanes in a direction are counted in 32 bits)
    DPEP_REQUIRE(num_sequences <= DPEP_MAX_SEQUENCES, "%s: num_sequences=%d is more than %d", what, num_sequences, DPEP_MAX_SEQUENCES);
    DPEP_REQUIRE(num_sequences >= 1 && (sequence_offsets != nullptr || num_sequences == 1), "%s: num_sequences=%d", what, num_sequences);
    DPEP_REQUIRE(losses != nullptr && counts != nullptr && tokens != nullptr && scratch != nullptr, "%s: a NULL buffer", what);
    return DPEP_OK;
}

}  // namespace

extern "C" {

int dpep_route(const dpep_router* r, const void* logits, const float* bias, const uint8_t* token_mask, int num_tokens, void* topk_idx,
               float* topk_weights, void* stream)
{
    if (int rc = check_router(r, num_tokens, "route"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(bias == nullptr || r->score == DPEP_SCORE_SIGMOID, "route: a bias needs sigmoid scores");
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(logits != nullptr && topk_idx != nullptr && topk_weights != nullptr, "route: a NULL buffer");
    Forward call = {};
    call.logits = logits;
    call.bias = bias;
    call.token_mask = token_mask;
    call.topk_idx = topk_idx;
    call.topk_weights = topk_weights;
    call.sequences = 1;
    return run_forward(r, call, num_tokens, true, false, nullptr, nullptr, nullptr, nullptr, stream, "route");
}

size_t dpep_balance_scratch_bytes(int num_experts, int num_tokens, int num_sequences)
{
    if (num_experts < 1 || num_experts > kMaxRouterExperts || num_tokens < 0 || num_tokens > DPEP_MAX_ROUTER_TOKENS || num_sequences < 1) return 0;
    return BalanceScratch(num_experts, num_tokens, num_sequences).bytes;
}

int dpep_balance_loss(const dpep_router* r, const void* logits, const void* topk_idx, int num_tokens, const int32_t* sequence_offsets, int num_sequences,
                      float* losses, int32_t* counts, int32_t* tokens, void* scratch, void* stream)
{
    if (int rc = check_router(r, num_tokens, "balance_loss"); rc != DPEP_OK) return rc;
    if (int rc = check_balance(r, num_tokens, sequence_offsets, num_sequences, losses, counts, tokens, scratch, "balance_loss"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(num_tokens == 0 || (logits != nullptr && topk_idx != nullptr), "balance_loss: a NULL buffer");
    Forward call = {};
    call.logits = logits;
    call.topk_idx = const_cast<void*>(topk_idx);
    call.offsets = sequence_offsets;
    call.sequences = num_sequences;
    return run_forward(r, call, num_tokens, false, true, losses, counts, tokens, scratch, stream, "balance_loss");
}

int dpep_route_balance(const dpep_router* r, const void* logits, const float* bias, const uint8_t* token_mask, int num_tokens, const int32_t* sequence_offsets,
                       int num_sequences, void* topk_idx, float* topk_weights, float* losses, int32_t* counts, int32_t* tokens, void* scratch, void* stream)
{
    if (int rc = check_router(r, num_tokens, "route_balance"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(bias == nullptr || r->score == DPEP_SCORE_SIGMOID, "route_balance: a bias needs sigmoid scores");
    if (int rc = check_balance(r, num_tokens, sequence_offsets, num_sequences, losses, counts, tokens, scratch, "route_balance"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(num_tokens == 0 || (logits != nullptr && topk_idx != nullptr && topk_weights != nullptr), "route_balance: a NULL buffer");
    Forward call = {};
    call.logits = logits;
    call.bias = bias;
    call.token_mask = token_mask;
    call.topk_idx = topk_idx;
    call.topk_weights = topk_weights;
    call.offsets = sequence_offsets;
    call.sequences = num_sequences;
    return run_forward(r, call, num_tokens, true, true, losses, counts, tokens, scratch, stream, "route_balance");
}

int dpep_router_backward(const dpep_router* r, const dpep_router_gradients* g, int num_tokens, void* stream)
{
    if (int rc = check_router(r, num_tokens, "router_backward"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(g != nullptr, "router_backward: gradients is NULL");
    DPEP_REQUIRE(g->grad_weights != nullptr || g->grad_losses != nullptr, "router_backward: neither grad_weights nor grad_losses is given");
    DPEP_REQUIRE(g->grad_losses == nullptr || (g->counts != nullptr && g->tokens != nullptr && g->num_sequences >= 1 &&
                                               (g->sequence_offsets != nullptr || g->num_sequences == 1)),
                 "router_backward: grad_losses needs the counts and tokens of its sequences");
    if (g->grad_losses != nullptr)
        if (int rc = check_routes(r, num_tokens, "router_backward"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(g->grad_weights == nullptr || !r->normalize || g->topk_weights != nullptr || num_tokens == 0, "router_backward: normalised weights are needed");
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(g->logits != nullptr && g->topk_idx != nullptr && g->grad_logits != nullptr, "router_backward: a NULL buffer");
    const bool balance = g->grad_losses != nullptr;
    const Backward call = {g->logits, g->topk_idx, g->topk_weights, g->grad_weights, g->sequence_offsets, balance ? g->counts : nullptr, g->tokens, g->grad_losses,
                           g->grad_logits, num_tokens, r->num_experts, r->num_topk, balance ? g->num_sequences : 1, router_chunk(num_tokens), r->normalize != 0,
                           r->index_bytes == 8, whole_pieces(r, g->logits, g->grad_logits), r->scale, 1.0f / r->scale};
    const int chunks = (num_tokens + call.chunk - 1) / call.chunk;
    with_variant(r, [&](auto v, auto type, auto sigmoid) {
        router_backward_kernel<v(), type(), sigmoid()><<<chunks, kRouterThreads, 0, static_cast<hipStream_t>(stream)>>>(call);
    });
    return launch_status("router_backward");
}

}  // extern "C"
