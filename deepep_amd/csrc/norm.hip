// Root-mean-square norm of the rows with the residual's addition and an output in 8 bits, its gradients, and tokens in 8-bit integers.
//
//   s = x, or type(x + residual);  rstd = (mean s^2 + eps)^-1/2;  v = s rstd w
//   grad_x = rstd (g w - xh c) + grad_stream, xh = s rstd, c = mean(g w xh);  grad_w[h] = sum_t g xh
//
// The norm is of s as it is stored: the backward, which reads the stored rows, is the gradient of exactly what the forward computed.
// The 8-bit codes are rounded from v in fp32, not from y: one rounding instead of two.
//
// All of it is bound by memory (forward: two rows in, two out; backward: two or three in, one out, and almost no arithmetic), so a row is read
// once and stays in registers from the sum of its squares to its last code.
#include <algorithm>

#include "common.h"
#include "mx.h"

#pragma clang fp contract(off)

namespace dpep {
namespace {

constexpr int kVec = 8;  // values of a row that a thread handles together

template <int kType>
struct Raw {
    u32x4 word[kType == DPEP_TYPE_F32 ? 2 : 1];
};
template <int kType>
__device__ __forceinline__ Raw<kType> load_raw(const void* base, size_t at)
{
    Raw<kType> r;
    if constexpr (kType == DPEP_TYPE_F32) {
        r.word[0] = load16(static_cast<const float*>(base) + at);
        r.word[1] = load16(static_cast<const float*>(base) + at + 4);
    } else {
        r.word[0] = load16(static_cast<const uint16_t*>(base) + at);
    }
    return r;
}
template <int kType>
__device__ __forceinline__ void widen(const Raw<kType>& r, float (&v)[kVec])
{
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        if constexpr (kType == DPEP_TYPE_F32) v[i] = __uint_as_float(r.word[i >> 2][i & 3]);
        else if constexpr (kType == DPEP_TYPE_BF16) v[i] = bf16_to_f32((r.word[0][i >> 1] >> (16 * (i & 1))) & 0xffffu);
        else v[i] = f16_to_f32((r.word[0][i >> 1] >> (16 * (i & 1))) & 0xffffu);
    }
}
template <int kType>
__device__ __forceinline__ Raw<kType> narrow(const float (&v)[kVec])
{
    Raw<kType> r;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        if constexpr (kType == DPEP_TYPE_F32) r.word[i >> 2][i & 3] = __float_as_uint(v[i]);
        else if (i % 2 == 0) r.word[0][i >> 1] = kType == DPEP_TYPE_BF16 ? pack_bf16x2(v[i], v[i + 1]) : pack_f16x2(v[i], v[i + 1]);
    }
    return r;
}
template <int kType>
__device__ __forceinline__ void store_raw(void* base, size_t at, const Raw<kType>& r)
{
    if constexpr (kType == DPEP_TYPE_F32) {
        *reinterpret_cast<u32x4*>(static_cast<float*>(base) + at) = r.word[0];
        *reinterpret_cast<u32x4*>(static_cast<float*>(base) + at + 4) = r.word[1];
    } else {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + at) = r.word[0];
    }
}
// The weight's values, of the rows' type or fp32.
template <int kType>
__device__ __forceinline__ void load_weight(const void* weight, bool wide, int at, float (&w)[kVec])
{
    if (wide) widen<DPEP_TYPE_F32>(load_raw<DPEP_TYPE_F32>(weight, at), w);
    else widen<kType>(load_raw<kType>(weight, at), w);
}

// Sum and maximum over lanes in a fixed order, by moves between the lanes' registers (an LDS permute a step costs 50 ns and more).
template <int kMove, int kRowMask = 0xf>
__device__ __forceinline__ uint32_t moved(uint32_t v)
{
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kMove, kRowMask, 0xf, false));
}
template <int kMove, int kRowMask = 0xf>
__device__ __forceinline__ float add_moved(float v)
{
    return v + __uint_as_float(moved<kMove, kRowMask>(__float_as_uint(v)));
}
// Of the wave; in every lane.
__device__ __forceinline__ float wave_sum(float v)
{
    v = add_moved<0x111>(v);  // row_shr:1, 2, 4, 8
    v = add_moved<0x112>(v);
    v = add_moved<0x114>(v);
    v = add_moved<0x118>(v);
    v = add_moved<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v = add_moved<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(v)), 63)));
}
// Of 4, 16 or 64 lanes next to one another; in each of them.
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v)
{
    static_assert(kLanes == 4 || kLanes == 16 || kLanes == 64);
    v = max(v, moved<0xb1>(v));  // quad_perm:[1,0,3,2], [2,3,0,1]
    v = max(v, moved<0x4e>(v));
    if constexpr (kLanes == 4) return v;
    v = max(v, moved<0x124>(v));  // row_ror:4, 8
    v = max(v, moved<0x128>(v));
    if constexpr (kLanes == 16) return v;
    v = max(v, moved<0x142, 0xa>(v));
    v = max(v, moved<0x143, 0xc>(v));
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
// The same over a workgroup.  `shared`: a word for each wave; the caller keeps two uses of it apart.
template <int kThreads>
__device__ __forceinline__ float block_sum(float v, float* shared)
{
    v = wave_sum(v);
    if constexpr (kThreads > kWave) {
        if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) v += shared[w];
    }
    return v;
}
template <int kThreads>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* shared)
{
    v = lanes_max<kWave>(v);
    if constexpr (kThreads > kWave) {
        if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) v = max(v, shared[w]);
    }
    return v;
}

// Magnitudes are compared as integers: a NaN's bits are above infinity's, so that it is not lost as fmaxf loses it.
__device__ __forceinline__ uint32_t magnitude(const float (&v)[kVec])
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

// 8 codes of a token's values, given the largest magnitude of the token.  Beside an infinity, whose own inverse is zero and would make a NaN of it, the others are zeros:
// 2^-130 takes it to 127 with its sign and the largest finite number to 1/4.
struct TokenScale {
    float inverse, scale;
    __device__ __forceinline__ explicit TokenScale(uint32_t largest)
    {
        const float m = __uint_as_float(max(largest, __float_as_uint(1e-20f)));
        inverse = largest == 0x7f800000u ? 0x1p-130f : (1.0f / m) * 127.0f;
        scale = m / 127.0f;
    }
    __device__ __forceinline__ u32x2 codes(const float (&v)[kVec]) const
    {
        u32x2 out = {0u, 0u};
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int q = static_cast<int>(fminf(fmaxf(rintf(v[i] * inverse), -127.0f), 127.0f));
            out[i >> 2] |= (static_cast<uint32_t>(q) & 0xffu) << (8 * (i & 3));
        }
        return out;
    }
};

// ---- forward -------------------------------------------------------------------------------------------------------------------
// One workgroup a row; thread i of chunk c has values (c * kThreads + i) * 8 and on, so that 16 lanes next to one another hold a block of
// 128 and 4 one of 32.  BF16 rows of 7168 with a residual: 16384 rows in 158 us (6.0 TB/s), 4096 with FP8 codes in 47 us (5.7 TB/s; a copy of 1 GiB
// runs at 5.1), one in 2.8 us, which is a launch, two trips to memory and two sums over the workgroup.
template <int kThreads, int kChunks, int kType>
__global__ __launch_bounds__(kThreads) void norm_kernel(const dpep_norm p)
{
    __shared__ float sums[kThreads / kWave];
    __shared__ uint32_t tops[kThreads / kWave];
    const int tid = threadIdx.x, hidden = p.hidden;
    const size_t row = static_cast<size_t>(blockIdx.x) * hidden;
    float v[kChunks][kVec], w[kChunks][kVec];
    Raw<kType> x[kChunks], r[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int at = (c * kThreads + tid) * kVec;
        if (at >= hidden) continue;
        x[c] = load_raw<kType>(p.x, row + at);
        if (p.residual != nullptr) r[c] = load_raw<kType>(p.residual, row + at);
    }
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int at = (c * kThreads + tid) * kVec;
        if (at >= hidden) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[c][i] = w[c][i] = 0.0f;
            continue;
        }
        load_weight<kType>(p.weight, p.weight_type == DPEP_TYPE_F32, at, w[c]);
        widen<kType>(x[c], v[c]);
        if (p.residual != nullptr) {
            float more[kVec];
            widen<kType>(r[c], more);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[c][i] += more[i];
            const Raw<kType> s = narrow<kType>(v[c]);
            store_raw<kType>(p.stream_out, row + at, s);
            widen<kType>(s, v[c]);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum += v[c][i] * v[c][i];
    }
    sum = block_sum<kThreads>(sum, sums);
    const float rstd = 1.0f / sqrtf(sum / static_cast<float>(hidden) + p.eps);
    if (p.rstd != nullptr && tid == 0) p.rstd[blockIdx.x] = rstd;
    uint32_t largest = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int at = (c * kThreads + tid) * kVec;
        const bool live = at < hidden;
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[c][i] = v[c][i] * rstd * w[c][i];
        if (live && p.y != nullptr) store_raw<kType>(p.y, row + at, narrow<kType>(v[c]));
        if (p.quantize == DPEP_QUANT_FP8) {
            if (c * kThreads * kVec >= hidden) continue;  // (the same for all lanes)
            const uint32_t block = lanes_max<16>(live ? magnitude(v[c]) : 0u);
            const float m = __uint_as_float(max(block, __float_as_uint(1e-4f)));
            const float inverse = (1.0f / m) * 448.0f;
            if (!live) continue;
            u32x2 codes;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                codes[i] = mx_pack4(v[c][4 * i] * inverse, v[c][4 * i + 1] * inverse, v[c][4 * i + 2] * inverse, v[c][4 * i + 3] * inverse);
            *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(p.codes) + row + at) = codes;
            if (at % 128 == 0) static_cast<float*>(p.scales)[static_cast<size_t>(blockIdx.x) * ((hidden + 127) / 128) + at / 128] = m / 448.0f;
        } else if (p.quantize == DPEP_QUANT_MXFP8) {
            if (c * kThreads * kVec >= hidden) continue;
            const uint32_t block = lanes_max<4>(live ? magnitude(v[c]) : 0u);
            const int byte = block >= 0x7f800000u ? 255 : mx_scale_byte(__uint_as_float(block));  // (255 is the format's NaN)
            if (!live) continue;
            u32x2 codes;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                codes[i] = mx_pack4(mx_scaled(v[c][4 * i], byte), mx_scaled(v[c][4 * i + 1], byte), mx_scaled(v[c][4 * i + 2], byte), mx_scaled(v[c][4 * i + 3], byte));
            *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(p.codes) + row + at) = codes;
            if (at % 32 == 0) static_cast<uint8_t*>(p.scales)[(row + at) / 32] = static_cast<uint8_t>(byte);
        } else if (live) {
            largest = max(largest, magnitude(v[c]));
        }
    }
    if (p.quantize == DPEP_QUANT_INT8) {
        const TokenScale token(block_max<kThreads>(largest, tops));
        if (tid == 0) static_cast<float*>(p.scales)[blockIdx.x] = token.scale;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int at = (c * kThreads + tid) * kVec;
            if (at < hidden) *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(p.codes) + row + at) = token.codes(v[c]);
        }
    }
}

// ---- tokens in 8-bit integers -----------------------------------------------------------------------------------------------------
// A row in a workgroup's registers, as in the norm.  100 FP16 rows of 2880: 2.6 us.
template <int kThreads, int kChunks, int kType>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const void* x, int k, uint8_t* codes, float* scales)
{
    __shared__ uint32_t tops[kThreads / kWave];
    const size_t row = static_cast<size_t>(blockIdx.x) * k;
    Raw<kType> raw[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int at = (c * kThreads + static_cast<int>(threadIdx.x)) * kVec;
        if (at < k) raw[c] = load_raw<kType>(x, row + at);
    }
    uint32_t largest = 0;
    float v[kVec];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        if ((c * kThreads + static_cast<int>(threadIdx.x)) * kVec >= k) continue;
        widen<kType>(raw[c], v);
        largest = max(largest, magnitude(v));
    }
    const TokenScale token(block_max<kThreads>(largest, tops));
    if (threadIdx.x == 0) scales[blockIdx.x] = token.scale;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int at = (c * kThreads + static_cast<int>(threadIdx.x)) * kVec;
        if (at >= k) continue;
        widen<kType>(raw[c], v);
        *reinterpret_cast<u32x2*>(codes + row + at) = token.codes(v);
    }
}
// Rows that do not fit: two passes, of which the second finds the row in the L2 (4380 BF16 rows of 14736: 52 us by two passes, 31 by one).
template <int kType>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(const void* x, int k, uint8_t* codes, float* scales)
{
    __shared__ uint32_t tops[256 / kWave];
    const size_t row = static_cast<size_t>(blockIdx.x) * k;
    uint32_t largest = 0;
    float v[kVec];
    for (int at = threadIdx.x * kVec; at < k; at += 256 * kVec) {
        widen<kType>(load_raw<kType>(x, row + at), v);
        largest = max(largest, magnitude(v));
    }
    const TokenScale token(block_max<256>(largest, tops));
    if (threadIdx.x == 0) scales[blockIdx.x] = token.scale;
    for (int at = threadIdx.x * kVec; at < k; at += 256 * kVec) {
        widen<kType>(load_raw<kType>(x, row + at), v);
        *reinterpret_cast<u32x2*>(codes + row + at) = token.codes(v);
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------
// A workgroup takes rows blockIdx.x, + gridDim.x, ...; the weight and its share of grad_weight stay in registers, and the next row is under way while
// one is worked on (without that a row's loads, its sum over the workgroup and its stores follow one another).  The share leaves as one row of
// `partial`.  16384 BF16 rows of 7168 with a gradient of the stream: 180 us (5.2 TB/s), and 5 for the sum of `partial`; 777 FP16 rows of 2880: 7.4 and 4.4.
template <int kThreads, int kChunks, int kType>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(const dpep_norm_gradients p, float* partial)
{
    __shared__ float sums[2][kThreads / kWave];
    const int tid = threadIdx.x, hidden = p.hidden;
    struct Row {
        Raw<kType> g[kChunks], s[kChunks], more[kChunks];
        float rstd;
    };
    const auto load = [&](int t) {
        Row r;
        const size_t row = static_cast<size_t>(t) * hidden;
        r.rstd = p.rstd[t];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int at = (c * kThreads + tid) * kVec;
            if (at >= hidden) continue;
            r.g[c] = load_raw<kType>(p.grad_y, row + at);
            r.s[c] = load_raw<kType>(p.stream, row + at);
            if (p.grad_stream != nullptr) r.more[c] = load_raw<kType>(p.grad_stream, row + at);
        }
        return r;
    };
    Row next = load(blockIdx.x);  // (there are no more workgroups than rows)
    float gw[kChunks][kVec] = {}, w[kChunks][kVec];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int at = (c * kThreads + tid) * kVec;
        if (at < hidden) load_weight<kType>(p.weight, p.weight_type == DPEP_TYPE_F32, at, w[c]);
    }
    int turn = 0;
    for (int t = blockIdx.x; t < p.num_tokens; t += gridDim.x, turn ^= 1) {
        const Row now = next;
        if (t < p.num_tokens - static_cast<int>(gridDim.x)) next = load(t + gridDim.x);
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            if ((c * kThreads + tid) * kVec >= hidden) continue;
            float gv[kVec], sv[kVec];
            widen<kType>(now.g[c], gv);
            widen<kType>(now.s[c], sv);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float hat = sv[i] * now.rstd, gh = gv[i] * hat;
                gw[c][i] += gh;
                sum += gh * w[c][i];
            }
        }
        const float mean = block_sum<kThreads>(sum, sums[turn]) / static_cast<float>(hidden);
        const size_t row = static_cast<size_t>(t) * hidden;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int at = (c * kThreads + tid) * kVec;
            if (at >= hidden) continue;
            float gv[kVec], sv[kVec], out[kVec];
            widen<kType>(now.g[c], gv);
            widen<kType>(now.s[c], sv);
#pragma unroll
            for (int i = 0; i < kVec; ++i) out[i] = now.rstd * (gv[i] * w[c][i] - sv[i] * now.rstd * mean);
            if (p.grad_stream != nullptr) {
                float mv[kVec];
                widen<kType>(now.more[c], mv);
#pragma unroll
                for (int i = 0; i < kVec; ++i) out[i] += mv[i];
            }
            store_raw<kType>(p.grad_x, row + at, narrow<kType>(out));
        }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int at = (c * kThreads + tid) * kVec;
        if (at < hidden) store_raw<DPEP_TYPE_F32>(partial, static_cast<size_t>(blockIdx.x) * hidden + at, narrow<DPEP_TYPE_F32>(gw[c]));
    }
}

// Columns of `partial` [rows,H] added up, 64 columns a workgroup: 64 rows at a time, four columns a lane.
__global__ __launch_bounds__(1024) void sum_partial_kernel(const float* partial, int rows, int hidden, float* out)
{
    __shared__ __attribute__((aligned(16))) float part[64][64];
    const int first = threadIdx.x / 16, at = threadIdx.x % 16 * 4, column = blockIdx.x * 64 + at;
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (column < hidden) {  // (H is a multiple of 8)
#pragma unroll 8
        for (int r = first; r < rows; r += 64) sum += *reinterpret_cast<const f32x4*>(partial + static_cast<size_t>(r) * hidden + column);
    }
    *reinterpret_cast<f32x4*>(&part[first][at]) = sum;
    __syncthreads();
    // 16 threads a column, four rows each, then the 16 of them in turn.
    const int mine = threadIdx.x / 16, group = threadIdx.x % 16;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v += part[group * 4 + i][mine];
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if (group == 0 && blockIdx.x * 64 + mine < hidden) out[blockIdx.x * 64 + mine] = v;
}

// Workgroups of the backward.  More of them have more loads under way, but each writes a row of `partial` that is read again: one to a compute unit for long rows, two
// for rows of up to 4096 values, four for up to 1024, more than one only where each then has four rows or more; up to 256 rows take a workgroup each (BF16, us with 256, 512 and 1024 workgroups: 9240 rows of 1024 33, 22, 20; of 2144 37, 29, 33; of
// 4096 46, 44, 48; of 7168 79, 82, 86; 777 of 2880 10.9, 12.1, 15).
inline int backward_groups(int tokens, int hidden)
{
    int groups = hidden <= 1024 ? 1024 : hidden <= 4096 ? 512 : 256;
    while (groups > 256 && tokens < 4 * groups) groups /= 2;
    return std::min(tokens, groups);
}

// The kernel for rows of `hidden` values: f(threads, chunks).  Few rows leave the machine empty and each is as quick as its longest thread; of many, four
// pieces a thread keep more loads under way.
template <class F>
void by_hidden(int tokens, int hidden, F f)
{
    if (tokens <= 256 && hidden > 256 * kVec) {
        if (hidden <= 512 * kVec) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 1>{});
        else if (hidden <= 1024 * kVec) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 1>{});
        else f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
    } else if (hidden <= 64 * kVec) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (hidden <= 256 * kVec) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    else if (hidden <= 512 * kVec) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (hidden <= 1024 * kVec) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
}
template <class F>
void by_type(int type, F f)
{
    if (type == DPEP_TYPE_F32) f(std::integral_constant<int, DPEP_TYPE_F32>{});
    else if (type == DPEP_TYPE_BF16) f(std::integral_constant<int, DPEP_TYPE_BF16>{});
    else f(std::integral_constant<int, DPEP_TYPE_F16>{});
}
inline bool is_type(int type) { return type == DPEP_TYPE_F32 || type == DPEP_TYPE_BF16 || type == DPEP_TYPE_F16; }
inline size_t bytes_of(int type) { return type == DPEP_TYPE_F32 ? 4 : 2; }

int check_rows(const char* what, int type, int weight_type, int tokens, int hidden)
{
    DPEP_REQUIRE(is_type(type), "%s: type=%d is not one of DPEP_TYPE_*", what, type);
    DPEP_REQUIRE(weight_type == type || weight_type == DPEP_TYPE_F32, "%s: weight_type=%d is neither the rows' type nor FP32", what, weight_type);
    DPEP_REQUIRE(tokens >= 0 && tokens <= DPEP_NORM_MAX_TOKENS, "%s: T=%d is not in [0, 2^23)", what, tokens);
    DPEP_REQUIRE(hidden >= 8 && hidden % 8 == 0 && hidden <= DPEP_NORM_MAX_HIDDEN, "%s: H=%d is not a multiple of 8 in [8, %d]", what, hidden, DPEP_NORM_MAX_HIDDEN);
    return DPEP_OK;
}

}  // namespace
}  // namespace dpep

using namespace dpep;

extern "C" {

int dpep_rms_norm(const dpep_norm* n, void* stream)
{
    DPEP_REQUIRE(n != nullptr, "rms_norm: NULL");
    if (int rc = check_rows("rms_norm", n->type, n->weight_type, n->num_tokens, n->hidden); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(n->quantize >= DPEP_QUANT_NONE && n->quantize <= DPEP_QUANT_INT8, "rms_norm: quantize=%d is not one of DPEP_QUANT_*", n->quantize);
    const int unit = n->quantize == DPEP_QUANT_NONE ? 8 : n->quantize == DPEP_QUANT_MXFP8 ? 32 : 16;
    DPEP_REQUIRE(n->hidden % unit == 0, "rms_norm: H=%d is not a multiple of %d", n->hidden, unit);
    DPEP_REQUIRE(n->eps >= 0.0f && n->eps <= 1.0f, "rms_norm: eps=%g is not in [0, 1]", static_cast<double>(n->eps));
    if (n->num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(n->x != nullptr && n->weight != nullptr && (n->residual == nullptr) == (n->stream_out == nullptr), "rms_norm: a NULL buffer");
    DPEP_REQUIRE((n->codes != nullptr) == (n->quantize != DPEP_QUANT_NONE) && (n->scales != nullptr) == (n->quantize != DPEP_QUANT_NONE),
                 "rms_norm: codes and scales belong to quantize");
    DPEP_REQUIRE(aligned16(n->x) && aligned16(n->residual) && aligned16(n->weight) && aligned16(n->stream_out) && aligned16(n->y) && aligned16(n->codes),
                 "rms_norm: a misaligned buffer");
    const size_t cells = static_cast<size_t>(n->num_tokens) * n->hidden, rows = cells * bytes_of(n->type), of_weight = n->hidden * bytes_of(n->weight_type);
    const size_t of_scales = n->quantize == DPEP_QUANT_FP8 ? static_cast<size_t>(n->num_tokens) * ((n->hidden + 127) / 128) * 4
                             : n->quantize == DPEP_QUANT_MXFP8 ? cells / 32 : static_cast<size_t>(n->num_tokens) * 4;
    const Span outputs[] = {{n->y, rows}, {n->rstd, static_cast<size_t>(n->num_tokens) * 4}, {n->codes, cells}, {n->scales, of_scales}};
    const Span inputs[] = {{n->x, rows}, {n->residual, rows}, {n->weight, of_weight}, {n->stream_out, rows}};
    DPEP_REQUIRE(apart(outputs, inputs), "rms_norm: an output overlaps an input or another output");
    DPEP_REQUIRE((n->stream_out == n->x || !overlap(n->stream_out, rows, n->x, rows)) && (n->stream_out == n->residual || !overlap(n->stream_out, rows, n->residual, rows)) &&
                     !overlap(n->stream_out, rows, n->weight, of_weight),
                 "rms_norm: stream_out overlaps an input");
    by_type(n->type, [&](auto type) {
        by_hidden(n->num_tokens, n->hidden, [&](auto threads, auto chunks) {
            norm_kernel<decltype(threads)::value, decltype(chunks)::value, decltype(type)::value>
                <<<n->num_tokens, decltype(threads)::value, 0, static_cast<hipStream_t>(stream)>>>(*n);
        });
    });
    return launch_status("rms_norm");
}

size_t dpep_rms_norm_backward_scratch_bytes(int num_tokens, int hidden)
{
    if (num_tokens < 0 || hidden < 0) return 0;
    return static_cast<size_t>(backward_groups(num_tokens, hidden)) * hidden * 4;
}

int dpep_rms_norm_backward(const dpep_norm_gradients* g, void* scratch, void* stream)
{
    DPEP_REQUIRE(g != nullptr, "rms_norm_backward: NULL");
    if (int rc = check_rows("rms_norm_backward", g->type, g->weight_type, g->num_tokens, g->hidden); rc != DPEP_OK) return rc;
    DPEP_REQUIRE(g->weight != nullptr && g->grad_weight != nullptr, "rms_norm_backward: a NULL buffer");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int groups = backward_groups(g->num_tokens, g->hidden);
    if (groups > 0) {
        DPEP_REQUIRE(g->grad_y != nullptr && g->stream != nullptr && g->rstd != nullptr && g->grad_x != nullptr && scratch != nullptr, "rms_norm_backward: a NULL buffer");
        DPEP_REQUIRE(aligned16(g->grad_y) && aligned16(g->stream) && aligned16(g->weight) && aligned16(g->grad_stream) && aligned16(g->grad_x) && aligned16(scratch),
                     "rms_norm_backward: a misaligned buffer");
        const size_t rows = static_cast<size_t>(g->num_tokens) * g->hidden * bytes_of(g->type), of_weight = g->hidden * bytes_of(g->weight_type);
        const Span written[] = {{g->grad_x, rows}, {g->grad_weight, g->hidden * 4ull}, {scratch, groups * (g->hidden * 4ull)}};
        const Span read[] = {{g->grad_x == g->grad_y ? nullptr : g->grad_y, rows}, {g->grad_x == g->grad_stream ? nullptr : g->grad_stream, rows}, {g->stream, rows},
                             {g->weight, of_weight}, {g->rstd, static_cast<size_t>(g->num_tokens) * 4}};
        DPEP_REQUIRE(apart(written, read), "rms_norm_backward: an output or scratch overlaps an input or one another");
        by_type(g->type, [&](auto type) {
            constexpr int kType = decltype(type)::value;
            float* const partial = static_cast<float*>(scratch);
            const int hidden = g->hidden;
            if (hidden <= 64 * kVec) norm_backward_kernel<64, 1, kType><<<groups, 64, 0, s>>>(*g, partial);
            else if (hidden <= 256 * kVec) norm_backward_kernel<256, 1, kType><<<groups, 256, 0, s>>>(*g, partial);
            else if (hidden <= 512 * kVec) norm_backward_kernel<512, 1, kType><<<groups, 512, 0, s>>>(*g, partial);
            else if (hidden <= 1024 * kVec) norm_backward_kernel<512, 2, kType><<<groups, 512, 0, s>>>(*g, partial);
            else norm_backward_kernel<1024, 2, kType><<<groups, 1024, 0, s>>>(*g, partial);
        });
        if (int rc = launch_status("rms_norm_backward"); rc != DPEP_OK) return rc;
    }
    sum_partial_kernel<<<(g->hidden + 63) / 64, 1024, 0, s>>>(static_cast<const float*>(scratch), groups, g->hidden, g->grad_weight);
    return launch_status("rms_norm_backward");
}

int dpep_quantize_tokens(const void* x, int type, int num_tokens, int k, int8_t* codes, float* scales, void* stream)
{
    DPEP_REQUIRE(is_type(type), "quantize_tokens: type=%d is not one of DPEP_TYPE_*", type);
    DPEP_REQUIRE(num_tokens >= 0 && num_tokens <= DPEP_W8_MAX_ROWS, "quantize_tokens: T=%d is not in [0, %d]", num_tokens, DPEP_W8_MAX_ROWS);
    DPEP_REQUIRE(k >= 16 && k % 16 == 0 && k <= DPEP_W8_MAX_K, "quantize_tokens: K=%d is not a multiple of 16 in [16, %d]", k, DPEP_W8_MAX_K);
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr && aligned16(x) && aligned16(codes), "quantize_tokens: a NULL or misaligned buffer");
    const size_t cells = static_cast<size_t>(num_tokens) * k, rows = cells * bytes_of(type);
    const Span written[] = {{codes, cells}, {scales, num_tokens * 4ull}}, read[] = {{x, rows}};
    DPEP_REQUIRE(apart(written, read), "quantize_tokens: an output overlaps x or the other output");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    uint8_t* const to = reinterpret_cast<uint8_t*>(codes);
    by_type(type, [&](auto t) {
        if (k <= DPEP_NORM_MAX_HIDDEN)
            by_hidden(num_tokens, k, [&](auto threads, auto chunks) {
                quantize_rows_kernel<decltype(threads)::value, decltype(chunks)::value, decltype(t)::value><<<num_tokens, decltype(threads)::value, 0, s>>>(x, k, to, scales);
            });
        else quantize_tokens_kernel<decltype(t)::value><<<num_tokens, 256, 0, s>>>(x, k, to, scales);
    });
    return launch_status("quantize_tokens");
}

}  // extern "C"
