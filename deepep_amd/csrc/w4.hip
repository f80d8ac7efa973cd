// Products of a few rows with matrices held in 4 bits with group scales: one matrix, and the experts of a routed layer.
//
//   W[n,k] = (q[n,k] - zero[n,k/G]) * scale[n,k/G],  y[m,n] = sum_k x[m,k] W[n,k]
//   experts: h = silu(W1g[e] x_t) * (W1u[e] x_t),  y_t = sum_s w_ts W2[e] h
#include "common.h"

#pragma clang fp contract(off)

namespace dpep {
namespace {

constexpr int kMaxRoutes = 2048;

// Expert ids of 8 or 4 bytes.
struct Ids {
    const void* ids;
    bool wide;
    int begin, local;
    // Local expert of a route, -1 if it has none here.
    __device__ __forceinline__ int operator[](int route) const
    {
        const long long e = (wide ? static_cast<const int64_t*>(ids)[route] : static_cast<const int32_t*>(ids)[route]) - static_cast<long long>(begin);
        return e >= 0 && e < local ? static_cast<int>(e) : -1;
    }
};

__device__ __forceinline__ float widen(uint32_t bits, bool half) { return half ? f16_to_f32(bits) : bf16_to_f32(bits); }
__device__ __forceinline__ uint16_t narrow(float v, bool half) { return static_cast<uint16_t>((half ? pack_f16x2(v, 0.0f) : pack_bf16x2(v, 0.0f)) & 0xffffu); }

// One row of a matrix times a vector, by a wave: every lane takes 32 values of k at a time.
template <class X>
__device__ float row_product(const dpep_w4& w, bool half, size_t row, const X* x, int lane)
{
    const uint8_t* const q = w.packed + row * (w.k / 2);
    const size_t groups = w.k / w.group;
    float sum = 0.0f;
    for (int k = lane * 32; k < w.k; k += kWave * 32) {
        const size_t g = row * groups + k / w.group;
        const float scale = widen(static_cast<const uint16_t*>(w.scales)[g], half), zero = w.zeros == nullptr ? 8.0f : static_cast<float>(w.zeros[g]);
        float part = 0.0f;
        for (int i = 0; i < 16; ++i) {
            const uint32_t both = q[k / 2 + i];
            float a, b;
            if constexpr (sizeof(X) == 4) {
                a = x[k + 2 * i];
                b = x[k + 2 * i + 1];
            } else {
                a = widen(x[k + 2 * i], half);
                b = widen(x[k + 2 * i + 1], half);
            }
            part = fmaf(static_cast<float>(both & 15u) - zero, a, part);
            part = fmaf(static_cast<float>(both >> 4) - zero, b, part);
        }
        sum = fmaf(part, scale, sum);
    }
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    return sum;
}

__global__ __launch_bounds__(256) void matvec_kernel(const dpep_w4 w, bool half, const uint16_t* x, uint16_t* y)
{
    const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6), m = blockIdx.y;
    if (n >= w.n) return;
    const float sum = row_product(w, half, n, x + static_cast<size_t>(m) * w.k, lane);
    if (lane == 0) y[static_cast<size_t>(m) * w.n + n] = narrow(sum, half);
}

__global__ __launch_bounds__(256) void gate_up_kernel(const dpep_w4 w, bool half, const uint16_t* x, const Ids ids, int topk, float* h)
{
    const int lane = threadIdx.x & 63, inter = w.n / 2, n = blockIdx.x * 4 + (threadIdx.x >> 6), route = blockIdx.y;
    const int e = ids[route];
    if (n >= inter || e < 0) return;
    const uint16_t* const row = x + static_cast<size_t>(route / topk) * w.k;
    const float gate = row_product(w, half, static_cast<size_t>(e) * w.n + n, row, lane);
    const float up = row_product(w, half, static_cast<size_t>(e) * w.n + inter + n, row, lane);
    if (lane == 0) h[static_cast<size_t>(route) * inter + n] = gate / (1.0f + expf(-gate)) * up;
}

__global__ __launch_bounds__(256) void down_kernel(const dpep_w4 w, bool half, const float* h, const Ids ids, const float* weights, int topk, uint16_t* y)
{
    const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6), token = blockIdx.y;
    if (n >= w.n) return;
    float sum = 0.0f;
    for (int s = 0; s < topk; ++s) {
        const int route = token * topk + s;
        const int e = ids[route];
        if (e < 0) continue;
        sum = fmaf(weights[route], row_product(w, half, static_cast<size_t>(e) * w.n + n, h + static_cast<size_t>(route) * w.k, lane), sum);
    }
    if (lane == 0) y[static_cast<size_t>(token) * w.n + n] = narrow(sum, half);
}

int check_w4(const dpep_w4* w, int type, const char* what)
{
    DPEP_REQUIRE(w != nullptr, "%s: weights is NULL", what);
    DPEP_REQUIRE(type == DPEP_TYPE_BF16 || type == DPEP_TYPE_F16, "%s: type=%d is neither BF16 nor FP16", what, type);
    DPEP_REQUIRE(w->n >= 1 && w->k >= 32, "%s: N=%d K=%d", what, w->n, w->k);
    DPEP_REQUIRE((w->group == 32 || w->group == 64 || (w->group >= 128 && w->group % 128 == 0)) && w->k % w->group == 0,
                 "%s: group=%d is not 32, 64 or a multiple of 128 that divides K=%d", what, w->group, w->k);
    DPEP_REQUIRE(w->packed != nullptr && w->scales != nullptr, "%s: a NULL buffer", what);
    DPEP_REQUIRE(aligned16(w->packed), "%s: packed is not 16-byte aligned", what);
    return DPEP_OK;
}

}  // namespace
}  // namespace dpep

using namespace dpep;

extern "C" {

int dpep_w4_matvec(const dpep_w4* w, int type, const void* x, int num_rows, void* y, void* stream)
{
    if (int rc = check_w4(w, type, "w4_matvec"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(num_rows >= 0 && num_rows <= 65535, "w4_matvec: num_rows=%d is not in [0, 65535]", num_rows);
    if (num_rows == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && y != nullptr && aligned16(x), "w4_matvec: a NULL or misaligned buffer");
    matvec_kernel<<<dim3((w->n + 3) / 4, num_rows), 256, 0, static_cast<hipStream_t>(stream)>>>(*w, type == DPEP_TYPE_F16, static_cast<const uint16_t*>(x),
                                                                                               static_cast<uint16_t*>(y));
    return launch_status("w4_matvec");
}

size_t dpep_w4_experts_scratch_bytes(int num_tokens, int num_topk, int hidden, int intermediate)
{
    if (num_tokens < 0 || num_topk < 1 || hidden < 1 || intermediate < 1) return 0;
    return static_cast<size_t>(num_tokens) * num_topk * intermediate * 4;
}

int dpep_w4_experts(const dpep_w4* gate_up, const dpep_w4* down, int type, const void* x, const void* topk_idx, int index_bytes, const float* topk_weights,
                    int num_tokens, int num_topk, int expert_begin, int num_local, void* y, void* scratch, void* stream)
{
    if (int rc = check_w4(gate_up, type, "w4_experts: gate_up"); rc != DPEP_OK) return rc;
    if (int rc = check_w4(down, type, "w4_experts: down"); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(gate_up->n == 2 * down->k && gate_up->k == down->n, "w4_experts: gate_up [%d,%d] and down [%d,%d] do not belong together", gate_up->n, gate_up->k,
                 down->n, down->k);
    DPEP_REQUIRE(num_tokens >= 0 && num_topk >= 1 && num_topk <= DPEP_MAX_TOPK && static_cast<long long>(num_tokens) * num_topk <= kMaxRoutes,
                 "w4_experts: T=%d K=%d: at most %d routes of at most %d slots a token", num_tokens, num_topk, kMaxRoutes, DPEP_MAX_TOPK);
    DPEP_REQUIRE(num_local >= 1 && num_local <= DPEP_MAX_LOCAL_EXPERTS && expert_begin >= 0, "w4_experts: num_local=%d expert_begin=%d", num_local, expert_begin);
    DPEP_REQUIRE(index_bytes == 4 || index_bytes == 8, "w4_experts: index_bytes=%d", index_bytes);
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && topk_idx != nullptr && topk_weights != nullptr && y != nullptr && scratch != nullptr && aligned16(x) && aligned16(scratch),
                 "w4_experts: a NULL or misaligned buffer");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool half = type == DPEP_TYPE_F16;
    float* const h = static_cast<float*>(scratch);
    const Ids ids = {topk_idx, index_bytes == 8, expert_begin, num_local};
    gate_up_kernel<<<dim3((down->k + 3) / 4, num_tokens * num_topk), 256, 0, s>>>(*gate_up, half, static_cast<const uint16_t*>(x), ids, num_topk, h);
    down_kernel<<<dim3((down->n + 3) / 4, num_tokens), 256, 0, s>>>(*down, half, h, ids, topk_weights, num_topk, static_cast<uint16_t*>(y));
    return launch_status("w4_experts");
}

}  // extern "C"
