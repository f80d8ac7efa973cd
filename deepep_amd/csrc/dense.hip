// The gated feed-forward block with its gradients, and products in 8-bit integers.
//
//   z = x Wgu^T = (g, u);  h = silu(g) u;  y = h Wd^T
//   dh = dy Wd;  dz = (dh u sg (1 + g (1 - sg)), dh g sg), sg = sigmoid(g);  dx = dz Wgu;  dWgu = dz^T x;  dWd = dy^T h
//   y[t,n] = a[t] b[n] sum_k x[t,k] w[n,k] in 8-bit integers
//
// All of them are products C[m,n] = sum_k A(m,k) B(n,k) of operands that hold k or m / n contiguously, with something done to a
// result before it is stored.
#include <algorithm>
#include <type_traits>

#include "common.h"

#pragma clang fp contract(off)

namespace dpep {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kInt8 = 100;  // beside DPEP_TYPE_*

template <int kType>
using Sum = std::conditional_t<kType == kInt8, i32x4, f32x4>;

template <int kType>
__device__ __forceinline__ Sum<kType> multiply(u32x4 a, u32x4 b, Sum<kType> c)
{
    if constexpr (kType == DPEP_TYPE_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (kType == DPEP_TYPE_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

template <int kType>
__device__ __forceinline__ u32x4 narrow8(const float (&v)[8])
{
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = kType == DPEP_TYPE_BF16 ? pack_bf16x2(v[2 * i], v[2 * i + 1]) : pack_f16x2(v[2 * i], v[2 * i + 1]);
    return out;
}
__device__ __forceinline__ void store_wide(float* to, const float (&v)[8])
{
    *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void load_wide(const float* from, float (&v)[8])
{
    const f32x4 a = *reinterpret_cast<const f32x4*>(from), b = *reinterpret_cast<const f32x4*>(from + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
}

// What becomes of results.  Each takes eight of them next to one another in a row; columns are a multiple of eight but for those of kScaled.
enum Finish {
    kStore,     // C rounded to the operands' type
    kGated,     // columns of gate and up together: h, and the products where they are kept
    kGradient,  // dh, with the kept products: dz and h
    kScaled,    // 8-bit integers' sums with the scales of row and column
};
struct Output {
    void* c;            // [M, ldc]
    float* kept;        // [M, 2 N]: gate, then up
    void* h;            // kGradient: [M, N]
    const float* row_scale;
    const float* column_scale;
    int type;           // of C where kScaled
};

__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }

template <int kType>
__device__ __forceinline__ void finish_gated(const Output& o, size_t m, int n, int columns, const float (&gate)[8], const float (&up)[8])
{
    if (o.kept != nullptr) {
        store_wide(o.kept + m * 2 * columns + n, gate);
        store_wide(o.kept + m * 2 * columns + columns + n, up);
    }
    float h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = gate[i] * sigmoid(gate[i]) * up[i];
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(o.c) + m * columns + n) = narrow8<kType>(h);
}

template <int kType, Finish kFinish>
__device__ __forceinline__ void finish(const Output& o, size_t m, int n, int columns, const float (&v)[8])
{
    if constexpr (kFinish == kStore) {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(o.c) + m * columns + n) = narrow8<kType>(v);
    } else if constexpr (kFinish == kGradient) {
        float gate[8], up[8], h[8], dg[8], du[8];
        load_wide(o.kept + m * 2 * columns + n, gate);
        load_wide(o.kept + m * 2 * columns + columns + n, up);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float share = sigmoid(gate[i]);
            h[i] = gate[i] * share * up[i];
            dg[i] = v[i] * up[i] * share * (1.0f + gate[i] * (1.0f - share));
            du[i] = v[i] * gate[i] * share;
        }
        uint16_t* const dz = static_cast<uint16_t*>(o.c) + m * 2 * columns + n;
        *reinterpret_cast<u32x4*>(dz) = narrow8<kType>(dg);
        *reinterpret_cast<u32x4*>(dz + columns) = narrow8<kType>(du);
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(o.h) + m * columns + n) = narrow8<kType>(h);
    } else if constexpr (kFinish == kScaled) {
        const float row = o.row_scale[m];
        const size_t at = m * columns + n;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (n + i >= columns) break;
            const float y = v[i] * row * o.column_scale[n + i];
            if (o.type == DPEP_TYPE_F32) static_cast<float*>(o.c)[at + i] = y;
            else static_cast<uint16_t*>(o.c)[at + i] = static_cast<uint16_t>(o.type == DPEP_TYPE_BF16 ? f32_to_bf16(y) : pack_f16x2(y, 0.0f) & 0xffffu);
        }
    }
}

// One product.  A is [M,K] (k_of_a contiguous) or [K,M], B [N,K] or [K,N]; kGated: B has gate rows, then up rows, of `columns` each.
struct Product {
    const void* a;
    const void* b;
    int m, columns, k;
    Output out;
};

// ---- a tile of 64 x 64 at a time, operands staged value by value ----------------------------------------------------------------
constexpr int kTile = 64, kStep = 64, kPitch = kStep + 16;

template <int kType, bool kTransA, bool kTransB, Finish kFinish>
__global__ __launch_bounds__(256) void product_kernel(const Product p)
{
    using Value = std::conditional_t<kType == kInt8, int8_t, uint16_t>;
    constexpr int kOfMfma = kType == kInt8 ? 64 : 32, kLane = kOfMfma / 4;  // values of k of an MFMA, of a lane
    constexpr int kWide = kFinish == kGated ? kTile / 2 : kTile;            // columns of the tile
    __shared__ __attribute__((aligned(16))) Value lds[2][kTile][kPitch];
    __shared__ __attribute__((aligned(16))) float result[kTile][kTile + 4];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int n_tiles = (p.columns + kWide - 1) / kWide;
    const int m0 = blockIdx.x / n_tiles * kTile, n0 = blockIdx.x % n_tiles * kWide;
    Sum<kType> acc[2][2] = {};
    for (int k0 = 0; k0 < p.k; k0 += kStep) {
        for (int i = tid; i < kTile * kStep; i += 256) {
            {
                const int row = kTransA ? i % kTile : i / kStep, at = kTransA ? i / kTile : i % kStep;
                const bool live = m0 + row < p.m && k0 + at < p.k;
                const size_t from = kTransA ? static_cast<size_t>(k0 + at) * p.m + m0 + row : static_cast<size_t>(m0 + row) * p.k + k0 + at;
                lds[0][row][at] = live ? static_cast<const Value*>(p.a)[from] : Value{0};
            }
            {
                const int row = kTransB ? i % kTile : i / kStep, at = kTransB ? i / kTile : i % kStep;
                const int column = n0 + row % kWide;
                const bool live = column < p.columns && k0 + at < p.k;
                const size_t n = static_cast<size_t>(kFinish == kGated && row >= kWide ? p.columns : 0) + column;
                const size_t from = kTransB ? static_cast<size_t>(k0 + at) * p.columns + n : n * p.k + k0 + at;
                lds[1][row][at] = live ? static_cast<const Value*>(p.b)[from] : Value{0};
            }
        }
        __syncthreads();
#pragma unroll
        for (int step = 0; step < kStep; step += kOfMfma)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = wave / 2 * 32 + i * 16 + lane % 16, column = wave % 2 * 32 + j * 16 + lane % 16, at = step + lane / 16 * kLane;
                    acc[i][j] = multiply<kType>(*reinterpret_cast<const u32x4*>(&lds[1][column][at]), *reinterpret_cast<const u32x4*>(&lds[0][row][at]), acc[i][j]);
                }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) result[wave / 2 * 32 + i * 16 + lane % 16][wave % 2 * 32 + j * 16 + lane / 16 * 4 + e] = static_cast<float>(acc[i][j][e]);
    __syncthreads();
    for (int i = tid; i < kTile * kWide / 8; i += 256) {
        const int row = i / (kWide / 8), at = i % (kWide / 8) * 8;
        if (m0 + row >= p.m || n0 + at >= p.columns) continue;
        float v[8];
        load_wide(&result[row][at], v);
        if constexpr (kFinish == kGated) {
            float up[8];
            load_wide(&result[row][kWide + at], up);
            finish_gated<kType>(p.out, m0 + row, n0 + at, p.columns, v, up);
        } else {
            finish<kType, kFinish>(p.out, m0 + row, n0 + at, p.columns, v);
        }
    }
}

template <int kType, bool kTransA, bool kTransB, Finish kFinish>
int launch(const Product& p, hipStream_t stream)
{
    if (p.m == 0 || p.columns == 0) return DPEP_OK;
    constexpr int kWide = kFinish == kGated ? kTile / 2 : kTile;
    const long long tiles = static_cast<long long>((p.m + kTile - 1) / kTile) * ((p.columns + kWide - 1) / kWide);
    DPEP_REQUIRE(tiles <= 0xffffff, "a product of %d x %d is too large", p.m, p.columns);
    product_kernel<kType, kTransA, kTransB, kFinish><<<static_cast<unsigned>(tiles), 256, 0, stream>>>(p);
    return launch_status("product");
}

int check_ffn(const dpep_ffn* f, const char* what, int tokens)
{
    DPEP_REQUIRE(f != nullptr, "%s: NULL", what);
    DPEP_REQUIRE(f->type == DPEP_TYPE_BF16 || f->type == DPEP_TYPE_F16, "%s: type=%d is neither BF16 nor FP16", what, f->type);
    DPEP_REQUIRE(f->hidden >= 8 && f->hidden % 8 == 0 && f->hidden <= DPEP_FFN_MAX_DIM && f->inter >= 8 && f->inter % 8 == 0 && f->inter <= DPEP_FFN_MAX_DIM,
                 "%s: H=%d and I=%d have to be multiples of 8 in [8, %d]", what, f->hidden, f->inter, DPEP_FFN_MAX_DIM);
    DPEP_REQUIRE(tokens >= 0 && tokens <= DPEP_FFN_MAX_TOKENS, "%s: T=%d is not in [0, %d]", what, tokens, DPEP_FFN_MAX_TOKENS);
    DPEP_REQUIRE(f->gate_up != nullptr && f->down != nullptr && aligned16(f->gate_up) && aligned16(f->down), "%s: a NULL or misaligned matrix", what);
    return DPEP_OK;
}
inline size_t whole(size_t bytes) { return (bytes + 255) & ~static_cast<size_t>(255); }

template <class F>
int by_type(int type, F f)
{
    return type == DPEP_TYPE_BF16 ? f(std::integral_constant<int, DPEP_TYPE_BF16>{}) : f(std::integral_constant<int, DPEP_TYPE_F16>{});
}

}  // namespace
}  // namespace dpep

using namespace dpep;

extern "C" {

size_t dpep_gated_ffn_scratch_bytes(int num_tokens, int hidden, int inter)
{
    if (num_tokens < 0 || hidden < 0 || inter < 0) return 0;
    return whole(static_cast<size_t>(num_tokens) * inter * 2);
}

int dpep_gated_ffn(const dpep_ffn* f, const void* x, int num_tokens, void* y, float* kept, void* scratch, void* stream)
{
    if (int rc = check_ffn(f, "gated_ffn", num_tokens); rc != DPEP_OK) return rc;
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && y != nullptr && scratch != nullptr && aligned16(x) && aligned16(y) && aligned16(kept) && aligned16(scratch),
                 "gated_ffn: a NULL or misaligned buffer");
    const size_t rows = static_cast<size_t>(num_tokens) * f->hidden * 2, half = static_cast<size_t>(f->hidden) * f->inter * 2, products = static_cast<size_t>(num_tokens) * f->inter * 8;
    DPEP_REQUIRE(!overlap(y, rows, x, rows) && !overlap(y, rows, f->gate_up, 2 * half) && !overlap(y, rows, f->down, half) && !overlap(y, rows, kept, products) &&
                     !overlap(kept, products, x, rows) && !overlap(kept, products, f->gate_up, 2 * half) && !overlap(kept, products, f->down, half),
                 "gated_ffn: an output overlaps an input");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return by_type(f->type, [&](auto type) {
        constexpr int kType = decltype(type)::value;
        Product p = {x, f->gate_up, num_tokens, f->inter, f->hidden, {}};
        p.out.c = scratch;
        p.out.kept = kept;
        if (int rc = launch<kType, false, false, kGated>(p, s); rc != DPEP_OK) return rc;
        p = {scratch, f->down, num_tokens, f->hidden, f->inter, {}};
        p.out.c = y;
        return launch<kType, false, false, kStore>(p, s);
    });
}

size_t dpep_gated_ffn_backward_scratch_bytes(int num_tokens, int hidden, int inter)
{
    if (num_tokens < 0 || hidden < 0 || inter < 0) return 0;
    return whole(static_cast<size_t>(num_tokens) * inter * 2) + whole(static_cast<size_t>(num_tokens) * inter * 4);
}

int dpep_gated_ffn_backward(const dpep_ffn* f, const void* grad_y, const void* x, const float* kept, int num_tokens, void* grad_x, void* grad_gate_up,
                            void* grad_down, void* scratch, void* stream)
{
    if (int rc = check_ffn(f, "gated_ffn_backward", num_tokens); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(grad_gate_up != nullptr && grad_down != nullptr && aligned16(grad_gate_up) && aligned16(grad_down), "gated_ffn_backward: a NULL or misaligned buffer");
    DPEP_REQUIRE(num_tokens == 0 || (grad_y != nullptr && x != nullptr && kept != nullptr && grad_x != nullptr && scratch != nullptr && aligned16(grad_y) && aligned16(x) &&
                                     aligned16(kept) && aligned16(grad_x) && aligned16(scratch)),
                 "gated_ffn_backward: a NULL or misaligned buffer");
    const size_t rows = static_cast<size_t>(num_tokens) * f->hidden * 2, half = static_cast<size_t>(f->hidden) * f->inter * 2, products = static_cast<size_t>(num_tokens) * f->inter * 8;
    const struct { const void* p; size_t bytes; } inputs[] = {{grad_y, rows}, {x, rows}, {kept, products}, {f->gate_up, 2 * half}, {f->down, half}},
                                                  outputs[] = {{grad_x, rows}, {grad_gate_up, 2 * half}, {grad_down, half}};
    for (const auto& out : outputs) {
        for (const auto& in : inputs) DPEP_REQUIRE(!overlap(out.p, out.bytes, in.p, in.bytes), "gated_ffn_backward: an output overlaps an input");
        for (const auto& other : outputs)
            DPEP_REQUIRE(&out == &other || !overlap(out.p, out.bytes, other.p, other.bytes), "gated_ffn_backward: two outputs overlap");
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    void* const h = scratch;
    void* const dz = static_cast<uint8_t*>(scratch) + whole(static_cast<size_t>(num_tokens) * f->inter * 2);
    return by_type(f->type, [&](auto type) {
        constexpr int kType = decltype(type)::value;
        Product p = {grad_y, f->down, num_tokens, f->inter, f->hidden, {}};
        p.out.c = dz;
        p.out.kept = const_cast<float*>(kept);
        p.out.h = h;
        if (int rc = launch<kType, false, true, kGradient>(p, s); rc != DPEP_OK) return rc;
        p = {dz, f->gate_up, num_tokens, f->hidden, 2 * f->inter, {}};
        p.out.c = grad_x;
        if (int rc = launch<kType, false, true, kStore>(p, s); rc != DPEP_OK) return rc;
        p = {dz, x, 2 * f->inter, f->hidden, num_tokens, {}};
        p.out.c = grad_gate_up;
        if (int rc = launch<kType, true, true, kStore>(p, s); rc != DPEP_OK) return rc;
        p = {grad_y, h, f->hidden, f->inter, num_tokens, {}};
        p.out.c = grad_down;
        return launch<kType, true, true, kStore>(p, s);
    });
}

size_t dpep_w8_matmul_scratch_bytes(int num_rows, int n, int k)
{
    (void)num_rows, (void)n, (void)k;
    return 0;
}

int dpep_w8_matmul(const dpep_w8* w, const int8_t* x, const float* x_scales, int num_rows, int type, void* y, void* scratch, void* stream)
{
    DPEP_REQUIRE(w != nullptr, "w8_matmul: weights is NULL");
    DPEP_REQUIRE(type == DPEP_TYPE_F32 || type == DPEP_TYPE_BF16 || type == DPEP_TYPE_F16, "w8_matmul: type=%d is not one of DPEP_TYPE_*", type);
    DPEP_REQUIRE(w->k >= 16 && w->k % 16 == 0 && w->k <= DPEP_W8_MAX_K, "w8_matmul: K=%d is not a multiple of 16 in [16, %d]", w->k, DPEP_W8_MAX_K);
    DPEP_REQUIRE(w->n >= 1 && w->n <= DPEP_W8_MAX_N, "w8_matmul: N=%d is not in [1, %d]", w->n, DPEP_W8_MAX_N);
    DPEP_REQUIRE(num_rows >= 0 && num_rows <= DPEP_W8_MAX_ROWS, "w8_matmul: T=%d is not in [0, %d]", num_rows, DPEP_W8_MAX_ROWS);
    DPEP_REQUIRE(w->codes != nullptr && w->scales != nullptr && aligned16(w->codes), "w8_matmul: a NULL or misaligned matrix");
    if (num_rows == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && x_scales != nullptr && y != nullptr && aligned16(x), "w8_matmul: a NULL or misaligned buffer");
    DPEP_REQUIRE(scratch != nullptr || dpep_w8_matmul_scratch_bytes(num_rows, w->n, w->k) == 0, "w8_matmul: scratch is NULL");
    const size_t results = static_cast<size_t>(num_rows) * w->n * (type == DPEP_TYPE_F32 ? 4 : 2);
    DPEP_REQUIRE(!overlap(y, results, x, static_cast<size_t>(num_rows) * w->k) && !overlap(y, results, x_scales, num_rows * 4ull) &&
                     !overlap(y, results, w->codes, static_cast<size_t>(w->n) * w->k) && !overlap(y, results, w->scales, w->n * 4ull),
                 "w8_matmul: y overlaps an input");
    Product p = {x, w->codes, num_rows, w->n, w->k, {}};
    p.out.c = y;
    p.out.row_scale = x_scales;
    p.out.column_scale = w->scales;
    p.out.type = type;
    return launch<kInt8, false, false, kScaled>(p, static_cast<hipStream_t>(stream));
}

}  // extern "C"
