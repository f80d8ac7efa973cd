// The gated feed-forward block with its gradients, and products in 8-bit integers.
//
//   z = x Wgu^T = (g, u);  h = silu(g) u;  y = h Wd^T
//   dh = dy Wd;  dz = (dh u sg (1 + g (1 - sg)), dh g sg), sg = sigmoid(g);  dx = dz Wgu;  dWgu = dz^T x;  dWd = dy^T h
//   y[t,n] = a[t] b[n] sum_k x[t,k] w[n,k] in 8-bit integers
//
// All of them are products C[m,n] = sum_k A(m,k) B(n,k) of operands that hold k or m / n contiguously, with something done to a
// result before it is stored.
#include <algorithm>
#include <cmath>
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

// What becomes of results.  Sums are in 32 bits until here.  h and dz are rounded to the operands' type, once each from 32 bits, because the matrix cores take 16-bit
// operands in the next product; what the backward needs of the products, g and u, is kept in FP32, so that dz is off by its own rounding alone.  Each takes eight of them next to one another in a row; columns are a multiple of eight but for those of kScaled.
enum Finish {
    kStore,     // C rounded to the operands' type
    kGated,     // columns of gate and up together: h, and the products where they are kept
    kGradient,  // dh, with the kept products: dz and h
    kScaled,    // 8-bit integers' sums with the scales of row and column
};
struct Output {
    void* c;            // [M, N], of kGradient dz [M, 2 N]
    float* kept;        // [M, 2 N]: gate, then up
    void* h;            // kGradient: [M, N]
    const float* row_scale;
    const float* column_scale;
    int type;           // of C where kScaled
};

// 1 / (1 + 2^(-g log2 e)) by the machine's own power and reciprocal, each good to a whole step, which is up to 2 x 2^-24 of a value.  The power's argument is off by 1.23 x 2^-24 of
// itself (its rounding, and that of the constant), so that the share is off by up to ((1.23 |g| + 2) (1 - share) + 3) 2^-24 of it, and is 0 below 2^-126: some 8 x 2^-24 from g = -2 on, 1.23 |g| + 5
// far below, while h and dz are rounded to 2^-8 or 2^-11.  (The library's exponential and division, off by a step or two, are some 25 instructions a value: dh of 2048 tokens, 2048 and
// 1024 values 25.6 us with them, 24.1 so.)
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g)); }

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

typedef u32x4 scattered __attribute__((aligned(1)));  // 16 bytes anywhere
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
        float y[8];
        if (n + 8 <= columns) {
            // Rows of any number of columns begin anywhere: the memory pipeline takes 16 bytes from any address.  (8192 x 4095 of k = 7168: 202 us instead of 248 by single values, 184 where the rows are aligned.)
            const scattered* const scales = reinterpret_cast<const scattered*>(o.column_scale + n);
            const f32x4 scale[2] = {__builtin_bit_cast(f32x4, u32x4(scales[0])), __builtin_bit_cast(f32x4, u32x4(scales[1]))};
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = v[i] * row * scale[i / 4][i % 4];
            if (o.type == DPEP_TYPE_F32) {
                scattered* const to = reinterpret_cast<scattered*>(static_cast<float*>(o.c) + at);
                to[0] = __builtin_bit_cast(u32x4, f32x4{y[0], y[1], y[2], y[3]});
                to[1] = __builtin_bit_cast(u32x4, f32x4{y[4], y[5], y[6], y[7]});
            } else {
                *reinterpret_cast<scattered*>(static_cast<uint16_t*>(o.c) + at) = o.type == DPEP_TYPE_BF16 ? narrow8<DPEP_TYPE_BF16>(y) : narrow8<DPEP_TYPE_F16>(y);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (n + i >= columns) break;
            const float one = v[i] * row * o.column_scale[n + i];
            if (o.type == DPEP_TYPE_F32) static_cast<float*>(o.c)[at + i] = one;
            else static_cast<uint16_t*>(o.c)[at + i] = static_cast<uint16_t>(o.type == DPEP_TYPE_BF16 ? f32_to_bf16(one) : pack_f16x2(one, 0.0f) & 0xffffu);
        }
    }
}

// One product.  A is [M,K] (k_of_a contiguous) or [K,M], B [N,K] or [K,N]; kGated: B has gate rows, then up rows, of `columns` each.
struct Product {
    const void* a;
    const void* b;
    int m, columns, k;
    Output out;
    // how it is cut up: tiles, parts of k of `part_steps` steps, their sums
    int m_tiles, n_tiles, parts, part_steps, pitch;
    int turned_a;  // A holds m contiguously (where the kernel does not say so)
    void* partial;
};

// ---- large tiles on the matrix cores ------------------------------------------------------------------------------------------------
// A workgroup of eight waves makes a tile of 256 x 256 results, or fewer, 128 bytes of k at a time ("step").  Both operands go from memory to LDS without
// passing registers, each in two halves of rows (columns) of the tile; with kGated the halves of B are the gate and the up rows of the same
// columns.  A wave takes 16 kRows rows and 32 columns of each half, so that a step is four products of a half of A with a half of B: (0,0), (0,1), (1,1), (1,0).
//
// Tiles of 256 x 256 take these two at a time ("phases").  The waves w and w + 4 share a SIMD and run half a phase apart: while one multiplies, the other reads the
// fragments of its next phase from LDS and asks for halves of later steps.  A phase of a wave is [read, ask, wait, barrier, multiply, barrier], and waves
// 4 .. 7 pass one barrier more at the start, waves 0 .. 3 at the end.
//   Phase 0 reads A0, B0 and B1 and asks for A1 of step k + 1, phase 1 reads A1 and asks for A0, B0 and B1 of step k + 2, into the place of step k's; there are two
//   buffers.  A wait covers what was asked for more than two phases ago (8 loads of a wave are later), and the wave's own reads.
//   Read after write: what a phase reads was asked for two phases before, every wave has waited for it one phase before, and a barrier that all waves pass after
//   that lies in between.
//   Write after read: a half is overwritten from the phase after the one that read it on, and a wave passes the barrier of its reading phase only when
//   its fragments are in its registers.
//
// In LDS a row of 128 bytes of k holds its 16-byte pieces c at place c ^ key(row), so that eight lanes that read the same piece of eight rows find them in
// different banks.  Operands that hold m or n contiguously lie in LDS as rows of k, 128 values wide, and are turned as they are read
// (ds_read_tr: 16 lanes read four rows); their pieces are spread by the row so that 32 lanes, eight rows, meet no bank twice.
//
// The matrix instruction takes B as its first operand, so that a lane's four results are four columns of one row.  The columns of a pair of
// instructions are dealt so that a lane ends up with eight next to one another: 16 bytes of 16-bit results.
//
// 8192 tokens, 7168 and 2048 values, BF16: 372 us for the gated product (1.29 PFLOP/s), 211 for the second (1.14), 213 for dh, 880 for the three of the backward
// (1.37); 8192 x 4096 of 7168 in 8-bit integers: 184 (2.6 POP/s).  Power bounds these: the clock falls to 1.7 GHz, and inputs of zeros take 0.83 of the time.
//
// Rows, columns and values of k that are not there are read as zero (the loads' own bounds check): a half's record ends with its last row, and pieces
// behind the last column or, in the last step, behind the last k have an offset that is nowhere.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int rsrc __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512;
constexpr int kStepBytes = 128;
constexpr uint32_t kNowhere = 0x80000000u;

// For all loads but the last kLoads and for what was read from LDS, and for the other waves.
template <int kLoads>
__device__ __forceinline__ void wait_and_meet()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLoads) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void meet()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// 16 bytes a lane from an operand straight into LDS, lane after lane from base + kAt on.
template <int kAt>
__device__ __forceinline__ void load_to_lds(rsrc from, uint32_t offset, uint32_t base)
{
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" ::"s"(base), "n"(kAt), "v"(offset), "s"(from) : "memory", "scc", "m0");
}
// One operand of a tile as the loads see it: halves of kRowsOfHalf rows (or columns), kPer loads a wave each.
template <bool kTrans, int kRowsOfHalf, bool kPaired>
struct Operand {
    static constexpr int kPer = kRowsOfHalf / 64;
    static constexpr int kBytes = kRowsOfHalf * kStepBytes;
    static_assert(kRowsOfHalf == 128 || kRowsOfHalf == 64);
    uint64_t base[2];                            // where the halves' next step begins
    int records[2];                              // and how many bytes there are
    uint32_t offset[kTrans ? 2 : 1][kPer];       // a lane's place in a half (of each half, where the columns that are there make a difference)
    uint64_t advance_bytes;
    int left;                                    // values of k that are left from the next step on

    static __device__ __forceinline__ int key(int row)
    {
        if constexpr (kTrans && kRowsOfHalf == 128) return kPaired ? (row & 3) << 2 | (row >> 3 & 1) : (row & 3) << 2 | (row >> 3 & 1) << 1;
        else if constexpr (kTrans) return kPaired ? (row >> 1 & 1) << 2 | (row >> 3 & 1) : (row >> 3 & 1) << 2 | (row >> 1 & 1) << 1;
        else return kPaired ? (row & 3) | (row >> 3 & 1) << 2 : row & 7;
    }
    // A lane's row of a half in load i, and its piece of that row.
    static __device__ __forceinline__ int row_of(int i, int wave, int lane)
    {
        if constexpr (kTrans) return (wave * kPer + i) * (512 / kRowsOfHalf) + lane / (kRowsOfHalf / 8);
        else return (wave * kPer + i) * 8 + lane / 8;
    }
    static __device__ __forceinline__ int piece_of(int i, int wave, int lane) { return (kTrans ? lane % (kRowsOfHalf / 8) : lane % 8) ^ key(row_of(i, wave, lane)); }

    // rows: of the operand's whole matrix; first[h]: its row (column) where half h begins; there[h]: rows (columns) from there on; k .. in values.
    template <int kValue>
    __device__ __forceinline__ void set(const void* matrix, int rows, const int (&first)[2], const int (&there)[2], int k_all, int k0, int k1, int wave, int lane)
    {
        const long long stride = static_cast<long long>(kTrans ? rows : k_all) * kValue;
        left = k1 - k0;
        advance_bytes = kTrans ? (kStepBytes / kValue) * stride : kStepBytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            base[h] = reinterpret_cast<uint64_t>(matrix) + (kTrans ? k0 * stride + static_cast<long long>(first[h]) * kValue
                                                                               : first[h] * stride + static_cast<long long>(k0) * kValue);
            records[h] = there[h] <= 0 ? 0 : kTrans ? 0x7fffffff : static_cast<int>(min(there[h], kRowsOfHalf) * stride);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int piece = piece_of(i, wave, lane);
                const uint32_t place = static_cast<uint32_t>(row_of(i, wave, lane) * stride) + piece * 16;
                if constexpr (kTrans) offset[h][i] = piece * (16 / kValue) < there[h] ? place : kNowhere;
                else offset[0][i] = place;
            }
        }
        limit<kValue>(wave, lane);
    }
    // Where the next step is the last one or none: what lies behind the end of k is nowhere.
    template <int kValue>
    __device__ __forceinline__ void limit(int wave, int lane)
    {
        if (left >= kStepBytes / kValue) return;
#pragma unroll
        for (int h = 0; h < (kTrans ? 2 : 1); ++h)
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if ((kTrans ? row_of(i, wave, lane) : piece_of(i, wave, lane) * (16 / kValue)) >= left) offset[h][i] = kNowhere;
    }
    // On to the next step, after both halves have been asked for.
    template <int kValue>
    __device__ __forceinline__ void advance(int wave, int lane)
    {
        base[0] += advance_bytes;
        base[1] += advance_bytes;
        left -= kStepBytes / kValue;
        limit<kValue>(wave, lane);
    }
    // Ask for half kHalf of the next step, to kAt behind `lds`, the wave's own place in a half.
    template <int kHalf, int kAt>
    __device__ __forceinline__ void ask(uint32_t lds) const
    {
        const rsrc from = {static_cast<int>(base[kHalf]), static_cast<int>(base[kHalf] >> 32), records[kHalf], 0x00020000};
        const uint32_t* const o = offset[kTrans ? kHalf : 0];
        load_to_lds<kAt>(from, o[0], lds);
        if constexpr (kPer == 2) load_to_lds<kAt + 1024>(from, o[1], lds);
    }
};

__device__ __forceinline__ s16x4 read_turned(const uint8_t* p)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}
// 8 values of k of a lane, from rows of k at p and, four rows of kBytes further, the other four.
template <int kBytes>
__device__ __forceinline__ u32x4 read_turned_pair(const uint8_t* p)
{
    const u32x2 a = __builtin_bit_cast(u32x2, read_turned(p)), b = __builtin_bit_cast(u32x2, read_turned(p + 4 * kBytes));
    return u32x4{a[0], a[1], b[0], b[1]};
}

// Which piece of work a workgroup takes: workgroups go round the eight dies, each of which gets neighbouring tiles, in blocks of four tiles of rows, so that
// its L2 serves the operands that its tiles share.
struct Place {
    int m, n, part;
};
__device__ __forceinline__ Place place_of(unsigned id, unsigned total, int m_tiles, int n_tiles)
{
    const unsigned die = id % 8, share = total / 8, more = total % 8;
    const unsigned at = die * share + min(die, more) + id / 8;
    const unsigned tiles = static_cast<unsigned>(m_tiles) * n_tiles, part = at / tiles, tile = at - part * tiles;
    const unsigned block = 4u * n_tiles, which = tile / block, in = tile - which * block, high = min(4u, m_tiles - which * 4);
    // (divisions leave the scalar registers; what follows from the place should not)
    return {__builtin_amdgcn_readfirstlane(static_cast<int>(which * 4 + in % high)), __builtin_amdgcn_readfirstlane(static_cast<int>(in / high)),
            __builtin_amdgcn_readfirstlane(static_cast<int>(part))};
}

// How a product is made: by a stream of B, or by tiles of 128 x 128 in a ring of five stages, the same in two stages, which leave room for a second workgroup on a
// compute unit, or 256 x 256 in two.
enum Way { kStream, kRing, kPairs, kLargeTiles };
template <Way kWay>
struct Shape {
    static constexpr bool kLarge = kWay == kLargeTiles;
    static constexpr int kTile = kLarge ? 256 : 128, kHalf = kTile / 2;
    static constexpr int kWavesN = kLarge ? 4 : 2, kRows = kLarge ? 4 : 1;  // waves across the columns, 32 of each half a wave; 16s of rows of each half a wave
    static constexpr int kStage = 4 * kHalf * kStepBytes, kStages = kWay == kRing ? 5 : 2;
    static constexpr int kWavesOfSimd = kWay == kPairs ? 4 : 2;
};

template <int kType, bool kTransA, bool kTransB, Finish kFinish, Way kWay>
__device__ __forceinline__ void make_tile(const Product& p, unsigned id, unsigned total, uint8_t* lds)
{
    using S = Shape<kWay>;
    constexpr int kValue = kType == kInt8 ? 1 : 2, kValues = kStepBytes / kValue;  // bytes of a value, values of a step
    constexpr int kHalf = S::kHalf, kRows = S::kRows, kWide = kFinish == kGated ? kHalf : 2 * kHalf;
    using A = Operand<kTransA, kHalf, false>;
    using B = Operand<kTransB, kHalf, true>;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wave_row = wave / S::kWavesN, wave_column = wave % S::kWavesN;
    const Place place = place_of(id, total, p.m_tiles, p.n_tiles);
    const int m0 = place.m * 2 * kHalf, n0 = place.n * kWide;
    const int k0 = min(p.k, place.part * p.part_steps * kValues), k1 = min(p.k, k0 + p.part_steps * kValues);
    const int steps = (k1 - k0 + kValues - 1) / kValues;

    A a;
    B b;
    {
        const int first[2] = {m0, m0 + kHalf}, there[2] = {p.m - m0, p.m - m0 - kHalf};
        a.template set<kValue>(p.a, p.m, first, there, p.k, k0, k1, wave, lane);
    }
    {
        const int second = kFinish == kGated ? p.columns + n0 : n0 + kHalf, columns = p.columns - n0;
        const int first[2] = {n0, second}, there[2] = {columns, kFinish == kGated ? columns : columns - kHalf};
        b.template set<kValue>(p.b, p.columns, first, there, p.k, k0, k1, wave, lane);
    }
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    const uint32_t a_base = lds0 + wave * (A::kBytes / 8), b_base = lds0 + wave * (B::kBytes / 8);

    // Where a lane reads its fragments: a place for each 16 rows (kTransA) or half step, as the key tells them apart.
    constexpr int kPlaces = kTransA ? kRows : 2, kBytesK = 2 * kHalf;  // (bytes of a row of k)
    int read_a[kPlaces], read_b[2];
    {
        const int r = lane % 16, group = lane / 16;
        if constexpr (kTransA) {
            const int row = 8 * group + r / 4, piece = wave_row * 2 * kRows + (r % 4) / 2;
#pragma unroll
            for (int i = 0; i < kPlaces; ++i) read_a[i] = row * kBytesK + ((piece + 2 * i) ^ A::key(row)) * 16 + (r % 2) * 8;
        } else {
            const int row = wave_row * 16 * kRows + r;
#pragma unroll
            for (int i = 0; i < kPlaces; ++i) read_a[i] = row * kStepBytes + ((4 * i + group) ^ A::key(row)) * 16;
        }
        if constexpr (kTransB) {
            // (of a pair of instructions the first takes the lower four columns of an even piece and the upper four of an odd one)
            const int row = 8 * group + r / 4, piece = wave_column * 4 + r % 4;
#pragma unroll
            for (int i = 0; i < 2; ++i) read_b[i] = row * kBytesK + (piece ^ B::key(row)) * 16 + ((i ^ r) & 1) * 8;
        } else {
            const int row = wave_column * 32 + 8 * (r / 4) + r % 4;
#pragma unroll
            for (int i = 0; i < 2; ++i) read_b[i] = row * kStepBytes + ((4 * i + group) ^ B::key(row)) * 16;
        }
    }
    Sum<kType> acc[2][2][kRows][2] = {};  // [half of A][half of B][16 rows][of a pair of instructions]
    const auto read_rows = [&](int at, u32x4 (&f)[kRows][2]) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if constexpr (kTransA) f[i][s] = read_turned_pair<kBytesK>(lds + read_a[i] + at + s * 32 * kBytesK);
                else f[i][s] = *reinterpret_cast<const u32x4*>(lds + read_a[s] + at + i * 16 * kStepBytes);
            }
    };
    const auto read_columns = [&](int at, u32x4 (&f)[2][2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if constexpr (kTransB) f[i][s] = read_turned_pair<kBytesK>(lds + read_b[i] + at + s * 32 * kBytesK);
                else f[i][s] = *reinterpret_cast<const u32x4*>(lds + read_b[s] + at + i * 4 * kStepBytes);
            }
    };
    const auto multiply_halves = [&](Sum<kType> (&sum)[kRows][2], const u32x4 (&fa)[kRows][2], const u32x4 (&fb)[2][2]) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int f = 0; f < 2; ++f) sum[i][f] = multiply<kType>(fb[f][s], fa[i][s], sum[i][f]);
    };
    constexpr std::integral_constant<int, 0> c0;
    constexpr std::integral_constant<int, 1> c1;

    if constexpr (S::kLarge) {
        // LDS: [half of A][buffer], [half of B][buffer], so that a lane's places in both buffers are within the reach of an instruction's own offset.
        constexpr auto a_at = [](int half, int buffer) { return (2 * half + buffer) * A::kBytes; };
        constexpr auto b_at = [](int half, int buffer) { return 4 * A::kBytes + (2 * half + buffer) * B::kBytes; };
#pragma unroll
        for (int i = 0; i < 2; ++i) read_b[i] += b_at(0, 0);
        u32x4 fa[kRows][2], fb[2][2][2];  // [.][half step]; [half][of a pair][half step]
        const auto multiply_phase = [&](auto half, auto first, auto second) {
            __builtin_amdgcn_s_setprio(1);
            multiply_halves(acc[half][first], fa, fb[first]);
            multiply_halves(acc[half][second], fa, fb[second]);
            __builtin_amdgcn_s_setprio(0);
            meet();
        };
        // A step whose operands lie in buffer `now`.
        const auto step = [&](auto now, auto other) {
            read_columns(b_at(0, now) - b_at(0, 0), fb[0]);
            read_rows(a_at(0, now), fa);
            read_columns(b_at(1, now) - b_at(0, 0), fb[1]);
            a.template ask<1, a_at(1, other)>(a_base);
            a.template advance<kValue>(wave, lane);
            wait_and_meet<8>();
            multiply_phase(c0, c0, c1);
            read_rows(a_at(1, now), fa);
            a.template ask<0, a_at(0, now)>(a_base);
            b.template ask<0, b_at(0, now)>(b_base);
            b.template ask<1, b_at(1, now)>(b_base);
            b.template advance<kValue>(wave, lane);
            wait_and_meet<8>();
            multiply_phase(c1, c1, c0);
        };
        a.template ask<0, a_at(0, 0)>(a_base);
        b.template ask<0, b_at(0, 0)>(b_base);
        b.template ask<1, b_at(1, 0)>(b_base);
        a.template ask<1, a_at(1, 0)>(a_base);
        a.template advance<kValue>(wave, lane);
        b.template advance<kValue>(wave, lane);
        a.template ask<0, a_at(0, 1)>(a_base);
        b.template ask<0, b_at(0, 1)>(b_base);
        b.template ask<1, b_at(1, 1)>(b_base);
        b.template advance<kValue>(wave, lane);
        wait_and_meet<8>();
        if (wave >= 4) meet();
        for (int k = 0; k < steps; k += 2) {  // (an odd number of steps gets one of zeros: a way out between the two costs registers)
            step(c0, c1);
            step(c1, c0);
        }
        if (wave < 4) meet();
    } else if constexpr (kWay == kPairs) {
        // While a step is read and multiplied the next one is asked for, into the place of the one before; the other workgroup of the compute unit has the matrix
        // cores while this one waits, and goes on while it begins or ends a tile.
        u32x4 fa[2][kRows][2], fb[2][2][2];  // [half][.][half step]
        const auto step = [&](int at, uint32_t to) {
            wait_and_meet<0>();
            read_rows(at, fa[0]);
            read_columns(at + 2 * A::kBytes, fb[0]);
            a.template ask<0, 0>(a_base + to);
            read_columns(at + 2 * A::kBytes + B::kBytes, fb[1]);
            b.template ask<0, 2 * A::kBytes>(b_base + to);
            read_rows(at + A::kBytes, fa[1]);
            b.template ask<1, 2 * A::kBytes + B::kBytes>(b_base + to);
            a.template ask<1, A::kBytes>(a_base + to);
            a.template advance<kValue>(wave, lane);
            b.template advance<kValue>(wave, lane);
            __builtin_amdgcn_s_setprio(1);
            multiply_halves(acc[0][0], fa[0], fb[0]);
            multiply_halves(acc[0][1], fa[0], fb[1]);
            multiply_halves(acc[1][1], fa[1], fb[1]);
            multiply_halves(acc[1][0], fa[1], fb[0]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
        };
        a.template ask<0, 0>(a_base);
        b.template ask<0, 2 * A::kBytes>(b_base);
        b.template ask<1, 2 * A::kBytes + B::kBytes>(b_base);
        a.template ask<1, A::kBytes>(a_base);
        a.template advance<kValue>(wave, lane);
        b.template advance<kValue>(wave, lane);
        for (int k = 0; k < steps; k += 2) {
            step(0, S::kStage);
            if (k + 1 < steps) step(S::kStage, 0);
        }
    } else {
        // What bounds this is L1: with the products left out a workgroup takes as long, with the reads from LDS left out too, without the loads 0.8 of it.  Some 100 lines of
        // 128 bytes are under way a compute unit, however far ahead they are asked for, and come after 670 cycles in the mean (512 tokens, 7168 to 2 x
        // 2048: 40 us, 14 TB/s from L2).
        // A ring of kStages steps: while a step is multiplied, the next one's fragments are read and the step kStages - 1 further on is asked for, into the place of
        // the one before, whose fragments are in every wave's registers by the barrier.
        constexpr int kLoads = 4, kStages = S::kStages;  // loads of a wave for a step
        const auto ask = [&](int stage) {
            const uint32_t to = stage * S::kStage;
            a.template ask<0, 0>(a_base + to);
            a.template ask<1, A::kBytes>(a_base + to);
            b.template ask<0, 2 * A::kBytes>(b_base + to);
            b.template ask<1, 2 * A::kBytes + B::kBytes>(b_base + to);
            a.template advance<kValue>(wave, lane);
            b.template advance<kValue>(wave, lane);
        };
        u32x4 fa[2][2][kRows][2], fb[2][2][2][2];  // [set][half][.][half step]
        const auto read = [&](int stage, auto set) {
            const int at = stage * S::kStage;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                read_rows(at + h * A::kBytes, fa[set][h]);
                read_columns(at + 2 * A::kBytes + h * B::kBytes, fb[set][h]);
            }
        };
        int reading = 1, asking = kStages - 1;  // stages
        const auto step = [&](auto now, auto other) {
            wait_and_meet<(kStages - 3) * kLoads>();
            const int at = reading * S::kStage;
            const uint32_t to = asking * S::kStage;
            read_rows(at, fa[other][0]);
            multiply_halves(acc[0][0], fa[now][0], fb[now][0]);
            a.template ask<0, 0>(a_base + to);
            __builtin_amdgcn_sched_barrier(0);
            read_columns(at + 2 * A::kBytes, fb[other][0]);
            multiply_halves(acc[0][1], fa[now][0], fb[now][1]);
            b.template ask<0, 2 * A::kBytes>(b_base + to);
            __builtin_amdgcn_sched_barrier(0);
            read_columns(at + 2 * A::kBytes + B::kBytes, fb[other][1]);
            multiply_halves(acc[1][1], fa[now][1], fb[now][1]);
            b.template ask<1, 2 * A::kBytes + B::kBytes>(b_base + to);
            __builtin_amdgcn_sched_barrier(0);
            read_rows(at + A::kBytes, fa[other][1]);
            reading = reading + 1 == kStages ? 0 : reading + 1;
            asking = asking + 1 == kStages ? 0 : asking + 1;
            multiply_halves(acc[1][0], fa[now][1], fb[now][0]);
            a.template ask<1, A::kBytes>(a_base + to);
            a.template advance<kValue>(wave, lane);
            b.template advance<kValue>(wave, lane);
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) ask(i);
        wait_and_meet<(kStages - 2) * kLoads>();
        read(0, c0);
        for (int k = 0; k < steps; k += 2) {
            step(c0, c1);
            if (k + 1 < steps) step(c1, c0);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (what was asked for past the end is in LDS before the workgroup gives it up)

    const int column = n0 + wave_column * 32 + lane / 16 * 8;
#pragma unroll
    for (int ha = 0; ha < 2; ++ha)
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int m = m0 + ha * kHalf + wave_row * 16 * kRows + i * 16 + lane % 16;
            if (m >= p.m) continue;
            Sum<kType> v[2][2];
#pragma unroll
            for (int hb = 0; hb < 2; ++hb)
#pragma unroll
                for (int f = 0; f < 2; ++f) v[hb][f] = kTransB && (lane / 16) % 2 == 1 ? acc[ha][hb][i][1 - f] : acc[ha][hb][i][f];
            if (p.parts > 1) {
                // Sums of a part of k, [part][m][columns, twice as many where kGated].
                constexpr int kTimes = kFinish == kGated ? 2 : 1;
                const size_t wide = static_cast<size_t>(kTimes) * p.pitch;
                uint32_t* const row = static_cast<uint32_t*>(p.partial) + (static_cast<size_t>(place.part) * p.m + m) * wide;
#pragma unroll
                for (int hb = 0; hb < 2; ++hb) {
                    const int n = kFinish == kGated ? column : column + hb * kHalf;
                    if (n >= p.columns) continue;
                    u32x4* const to = reinterpret_cast<u32x4*>(row + (kFinish == kGated ? hb * static_cast<size_t>(p.pitch) : 0) + n);
                    to[0] = __builtin_bit_cast(u32x4, v[hb][0]);
                    to[1] = __builtin_bit_cast(u32x4, v[hb][1]);
                }
                continue;
            }
            float wide[2][8];
#pragma unroll
            for (int hb = 0; hb < 2; ++hb)
#pragma unroll
                for (int e = 0; e < 8; ++e) wide[hb][e] = static_cast<float>(v[hb][e / 4][e % 4]);
            if constexpr (kFinish == kGated) {
                if (column < p.columns) finish_gated<kType>(p.out, m, column, p.columns, wide[0], wide[1]);
            } else {
#pragma unroll
                for (int hb = 0; hb < 2; ++hb) {
                    const int n = column + hb * kHalf;
                    if (n < p.columns) finish<kType, kFinish>(p.out, m, n, p.columns, wide[hb]);
                }
            }
        }
}

template <int kType, bool kTransA, bool kTransB, Finish kFinish, Way kWay>
__global__ __launch_bounds__(kThreads, Shape<kWay>::kWavesOfSimd) void tile_kernel(const Product p)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Shape<kWay>::kStages * Shape<kWay>::kStage];
    make_tile<kType, kTransA, kTransB, kFinish, kWay>(p, blockIdx.x, gridDim.x, lds);
}

// Three products that do not wait for one another in one launch: workgroups of the next fill up the compute units that the last tiles of one leave idle.
// B holds n contiguously in all of them, A m in some.
// (What is picked out of the arguments by a computed index is whole words at whole words' distances: a byte for each product among them made
// the compiler take addresses that are no multiples of four into scalar loads, which ignore the lowest two bits of each part of an address.)
struct Products {
    Product of[3];
    unsigned begin[4];  // a product's first workgroup
};
static_assert(std::is_same_v<decltype(Product::turned_a), int> && sizeof(Product) % 8 == 0 && sizeof(Products) == 3 * sizeof(Product) + 4 * sizeof(unsigned),
              "what is picked by a computed index is whole words, and nothing lies beside the products and their begins");
template <int kType, Way kWay>
__global__ __launch_bounds__(kThreads, Shape<kWay>::kWavesOfSimd) void products_kernel(const Products p)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Shape<kWay>::kStages * Shape<kWay>::kStage];
    const int which = blockIdx.x < p.begin[1] ? 0 : blockIdx.x < p.begin[2] ? 1 : 2;
    const unsigned id = blockIdx.x - p.begin[which], total = p.begin[which + 1] - p.begin[which];
    if (p.of[which].turned_a != 0) make_tile<kType, true, true, kStore, kWay>(p.of[which], id, total, lds);
    else make_tile<kType, false, true, kStore, kWay>(p.of[which], id, total, lds);
}

// The parts of k added up, and what becomes of the sums.
template <int kType, Finish kFinish>
__global__ __launch_bounds__(256) void join_kernel(const Product p)
{
    constexpr int kTimes = kFinish == kGated ? 2 : 1;
    const size_t wide = static_cast<size_t>(kTimes) * p.pitch;
    const int pieces = p.pitch / 8;
    const size_t at = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    const size_t m = at / pieces;
    const int n = static_cast<int>(at - m * pieces) * 8;
    if (m >= static_cast<size_t>(p.m)) return;
    float v[kTimes][8];
#pragma unroll
    for (int t = 0; t < kTimes; ++t) {
        Sum<kType> sum[2] = {};
#pragma unroll 8
        for (int part = 0; part < p.parts; ++part) {
            const u32x4* const from = reinterpret_cast<const u32x4*>(static_cast<const uint32_t*>(p.partial) + (static_cast<size_t>(part) * p.m + m) * wide +
                                                                     static_cast<size_t>(t) * p.pitch + n);
            sum[0] += __builtin_bit_cast(Sum<kType>, from[0]);
            sum[1] += __builtin_bit_cast(Sum<kType>, from[1]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[t][e] = static_cast<float>(sum[e / 4][e % 4]);
    }
    if constexpr (kFinish == kGated) finish_gated<kType>(p.out, m, n, p.columns, v[0], v[1]);
    else finish<kType, kFinish>(p.out, m, n, p.columns, v[0]);
}

// ---- few rows: a stream of B ------------------------------------------------------------------------------------------------------
// For few rows of A the time is that of reading B.  A workgroup makes kGroups times 16 columns (kGated: 8 of gate and the same 8 of up) for up to 16 kBlocks rows; its eight waves take
// every eighth line of 128 bytes of k, and their sums meet in LDS at the end.  Each wave has a ring of its own in LDS, into which its lines of B and A
// go straight from memory, 8 rows of whole lines a load, and waits for nobody else on the way.  (Read to registers in the matrix instruction's own order a load of
// A touches 64 lines instead of 8: 64 rows of 7168, 4096 columns took 37 us by that.)
// One token: 7168 to 2 x 2048 in BF16 (59 MB) 12.0 us, 2048 to 7168 (29 MB) 7.3, 7168 to 4096 in 8 bits (29 MB) 7.6, where an empty kernel takes 2 to 3.
template <int kType, Finish kFinish, int kGroups, int kBlocks, int kStages>
__global__ __launch_bounds__(kThreads, 2) void stream_kernel(const Product p)
{
    constexpr int kValue = kType == kInt8 ? 1 : 2, kWaves = kThreads / kWave;
    constexpr int kLoadsB = 2 * kGroups, kLoads = kLoadsB + 2 * kBlocks, kStage = kLoads * 1024;  // of a wave for a line
    constexpr int kWide = kGroups * (kFinish == kGated ? 8 : 16);                                 // columns of the result
    static_assert(kLoads >= 4 && kLoads <= 10);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves * kStages * kStage];
    static_assert(sizeof(lds) >= kWaves * kGroups * kBlocks * 1024);
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n0 = blockIdx.x * kWide, m0 = blockIdx.y * 16 * kBlocks, rows = min(16 * kBlocks, p.m - m0);
    const int k_bytes = p.k * kValue, lines = (k_bytes + kStepBytes - 1) / kStepBytes;
    // 8 rows a load; what lies behind a load's last row is read as zero.  (8 rows are less than 2^31 bytes.)
    uint64_t base[kLoads];
    int records[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const bool of_b = j < kLoadsB;
        const int n = n0 + 8 * (kFinish == kGated ? j / 2 : j), in_a = (j - kLoadsB) * 8;
        const int row = of_b ? (kFinish == kGated && j % 2 == 1 ? p.columns : 0) + n : m0 + in_a, there = min(8, of_b ? p.columns - n : rows - in_a);
        base[j] = reinterpret_cast<uint64_t>(of_b ? p.b : p.a) + static_cast<uint64_t>(row) * k_bytes;
        records[j] = __builtin_amdgcn_readfirstlane(max(there, 0)) * k_bytes;  // (a number between two bounds comes from a vector instruction)
    }
    // Lane l loads a piece of row l / 8, which lies in LDS where the pieces of eight rows that are read together meet no bank twice.
    const int piece = lane % 8 ^ lane / 8;
    uint32_t at = wave * kStepBytes + piece * 16;  // in k, bytes
    const uint32_t row_at = lane / 8 * k_bytes;
    const uint32_t mine = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + wave * kStages * kStage;
    const auto from = [&](int j) { return rsrc{static_cast<int>(base[j]), static_cast<int>(base[j] >> 32), records[j], 0x00020000}; };
    const auto ask = [&](int stage) {
        const uint32_t place = at < static_cast<uint32_t>(k_bytes) ? row_at + at : kNowhere, to = mine + stage * kStage;
        load_to_lds<0>(from(0), place, to);
        load_to_lds<1024>(from(1), place, to);
        load_to_lds<2048>(from(2), place, to);
        load_to_lds<3 * 1024>(from(3), place, to);
        if constexpr (kLoads >= 6) {
            load_to_lds<4096>(from(4), place, to);
            load_to_lds<5120>(from(5), place, to);
        }
        if constexpr (kLoads >= 8) {
            load_to_lds<6144>(from(6), place, to);
            load_to_lds<7168>(from(7), place, to);
        }
        if constexpr (kLoads >= 10) {
            load_to_lds<8192>(from(8), place, to);
            load_to_lds<9216>(from(9), place, to);
        }
        at += kWaves * kStepBytes;
    };
    int read_at[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) read_at[s] = wave * kStages * kStage + lane % 16 * kStepBytes + ((4 * s + lane / 16) ^ (lane & 7)) * 16;
    Sum<kType> acc[kGroups][kBlocks] = {};
#pragma unroll
    for (int i = 0; i < kStages; ++i) ask(i);
    int stage = 0;
    for (int line = wave; line < lines; line += kWaves) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * kLoads) : "memory");
        u32x4 b[kGroups][2], a[kBlocks][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) b[g][s] = *reinterpret_cast<const u32x4*>(lds + read_at[s] + stage * kStage + 2048 * g);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) a[i][s] = *reinterpret_cast<const u32x4*>(lds + read_at[s] + stage * kStage + 2048 * (kGroups + i));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the stage is read, and may be asked for again)
        __builtin_amdgcn_sched_barrier(0);
        ask(stage);
        stage = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) acc[g][i] = multiply<kType>(b[g][s], a[i][s], acc[g][i]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    // Lane (q, r) has results 4 q .. 4 q + 3 of row r: sums[wave][group][block][row][16].
    uint32_t(*const sums)[kGroups][kBlocks][16][16] = reinterpret_cast<uint32_t(*)[kGroups][kBlocks][16][16]>(lds);
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) *reinterpret_cast<u32x4*>(&sums[wave][g][i][lane % 16][lane / 16 * 4]) = __builtin_bit_cast(u32x4, acc[g][i]);
    __syncthreads();
    const int m = threadIdx.x % (16 * kBlocks), octet = threadIdx.x / (16 * kBlocks);
    if (octet >= kWide / 8 || m >= rows) return;
    const auto total = [&](int group, int o, float (&v)[8]) {
        Sum<kType> sum[2] = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) sum[h] += __builtin_bit_cast(Sum<kType>, *reinterpret_cast<const u32x4*>(&sums[w][group][m / 16][m % 16][8 * o + 4 * h]));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(sum[e / 4][e % 4]);
    };
    const int n = n0 + 8 * octet;
    if (n >= p.columns) return;
    float v[8];
    if constexpr (kFinish == kGated) {
        float up[8];
        total(octet, 0, v);
        total(octet, 1, up);
        finish_gated<kType>(p.out, m0 + m, n, p.columns, v, up);
    } else {
        total(octet / 2, octet % 2, v);
        finish<kType, kFinish>(p.out, m0 + m, n, p.columns, v);
    }
}

constexpr long long kMostWorkgroups = 0x7fffff;  // of kThreads: a grid has less than 2^32 threads

// How a product is cut up, k into parts whose sums another kernel adds up.
struct Cut {
    Way way;
    int m_tiles, n_tiles, parts, part_steps;
    size_t bytes;  // of the parts' sums
    double us;
};
// The quickest by what was measured on 256 compute units.  Where all of them are at work a step of a large tile takes 1.5 us, of one in the ring 0.58, and of two that share a
// compute unit 0.92, with 5, 4 and 4.5 us around a tile's steps; a last round of pairs takes 0.75 of a whole one with no more than one tile a compute unit, 0.85 and up
// with more.  So pairs win from one to about two and a half tiles of 128 a compute unit, and where k is short (8-bit integers, 400 tiles, 23 steps: 31 us by the
// ring, 25 by pairs, 39 by large tiles; 256 tiles, 56 steps: 34, 43, 67; 1024 tiles, 56 steps: 126, 108, 88).
// Joining parts takes 3.5 us and 0.2 a part, and 2 ps for each of the 4-byte sums, written and read.  A round of 256 workgroups of a stream takes 3 us and what one
// reads of B and of up to 64 rows of A, at 62 bytes / ns; up to 16 rows, whose rounds run into one another, 3 us once and 0.35 for each 256 workgroups (8-bit, 6 rows of 432 to 62901: 22.9 us by 3932 short
// ones, 9.9 by pairs).  Beside that counts 0.4 of the time of reading B from memory.
inline double tile_us(Way way, int steps) { return way == kLargeTiles ? 10 + 1.45 * steps : way == kRing ? 4 + 0.58 * steps : 4.5 + 0.92 * steps; }
// Groups of 16 columns of a stream's workgroup.  Two read A half as often: for more tiles than compute units, and for up to 16 rows if they then fit one round; above that, two
// workgroups on a compute unit, with rings of two stages, end more evenly.  (16-bit, 14 rows of 6544 to 2 x 3304 and back, 413 and 409 tiles: 36 us by twos, 40 by ones; 24 rows, 7168
// to 2 x 2048: 27, 30; 8-bit, 3 rows of 15440 to 9681, 606 tiles: 42, 34.)
inline int stream_groups(int m, int n_tiles) { return n_tiles <= 256 || m > 32 || (m <= 16 && n_tiles > 512) ? 1 : 2; }
struct Stream {
    int groups, blocks, stages;
};
inline Stream stream_of(int m, int n_tiles)
{
    const int groups = stream_groups(m, n_tiles);
    if (m <= 16) return {groups, 1, groups == 2 ? 3 : n_tiles <= 256 ? 5 : 2};
    if (m <= 32) return {groups, 2, groups == 2 ? 2 : 3};
    return {1, 4, 2};
}
inline double join_us(int parts, size_t bytes) { return 3.5 + 0.2 * parts + 0.5e-6 * static_cast<double>(bytes); }
inline int at_once(Way way) { return way == kPairs ? 512 : 256; }
// No tiles are quicker than memory, which gives 5.8 MB / us, 2 us after the start, where every place for a workgroup is taken, and as much less as the rounds leave free, to half of it.  (The steps' costs above are those of operands
// that L2 holds for many tiles; of few rows every byte of B comes from memory.  8-bit, 4 rows of 28672 to 8192: 59 us by the pairs that the steps alone would choose, 43 by a stream; 1 row of 4096
// to 128256 114 and 95; 16-bit, 8 rows of 18432 to 7168 156 and 138.  1975 products of 1 to 2500 rows, every way timed: the chosen one is 1.8 % above the quickest in the mean; without this and the cost of a stream's
// workgroups 3.5.)
inline double memory_us(Way way, long long workgroups, double bytes)
{
    const double rounds = static_cast<double>(workgroups) / at_once(way);
    return workgroups == 0 ? 0 : 2 + bytes / 5.8e6 * std::min(2.0, std::ceil(rounds) / rounds);
}
inline double rounds_of(Way way, long long tiles)
{
    const long long whole = tiles / at_once(way), rest = tiles % at_once(way);
    if (rest == 0) return static_cast<double>(whole);
    return static_cast<double>(whole) + (way != kPairs ? 1.0 : rest <= 256 ? 0.75 : 0.7 + 0.3 * static_cast<double>(rest) / 512);
}
Cut cut_of(int m, int columns, int k_bytes, bool gated, bool turned)
{
    const int steps = std::max(1, (k_bytes + kStepBytes - 1) / kStepBytes), times = gated ? 2 : 1;
    const double needed = (static_cast<double>(columns) * times + m) * k_bytes + 2.0 * m * columns;  // both operands and 16-bit results
    Cut best = {};
    if (!turned) {
        const int n_tiles = (columns * times + 15) / 16, m_tiles = (m + 63) / 64, groups = stream_groups(m, n_tiles);
        const double workgroups = static_cast<double>((n_tiles + groups - 1) / groups) * m_tiles, read = static_cast<double>(16 * groups + std::min(m, 64)) * k_bytes / 62e3;
        const double rounds = m <= 16 && groups == 1 ? 3 + std::max(1.0, workgroups / 256) * read + 0.35 * workgroups / 256 : std::ceil(workgroups / 256) * (3 + read);
        best = {kStream, m_tiles, n_tiles, 1, steps, 0, 0.5 + rounds + 0.4 * columns * times * static_cast<double>(k_bytes) / 5.5e6};
    }
    for (const Way way : {kRing, kPairs, kLargeTiles}) {
        const int tile = way == kLargeTiles ? 256 : 128, wide = tile / times;
        const int m_tiles = (m + tile - 1) / tile, n_tiles = (columns + wide - 1) / wide;
        for (int wanted = 1; wanted <= 16; ++wanted) {
            const int part_steps = (steps + wanted - 1) / wanted, parts = (steps + part_steps - 1) / part_steps;
            const long long workgroups = static_cast<long long>(m_tiles) * n_tiles * parts;
            if (parts != wanted || workgroups > kMostWorkgroups) continue;
            const double rounds = rounds_of(way, workgroups);
            const size_t bytes = parts == 1 ? 0 : static_cast<size_t>(parts) * m * ((columns + 7) / 8 * 8) * times * 4;
            const double us = std::max(rounds * tile_us(way, part_steps), memory_us(way, workgroups, needed + bytes)) + (parts == 1 ? 0 : join_us(parts, bytes));
            if (best.parts == 0 || us < best.us) best = {way, m_tiles, n_tiles, parts, part_steps, bytes, us};
        }
    }
    return best;
}

inline Product cut_up(Product p, const Cut& c, void* partial)
{
    p.m_tiles = c.m_tiles;
    p.n_tiles = c.n_tiles;
    p.parts = c.parts;
    p.part_steps = c.part_steps;
    p.pitch = (p.columns + 7) / 8 * 8;
    p.partial = partial;
    return p;
}
// The sums of a product's parts, if it has any.
template <int kType, Finish kFinish>
int join(const Product& p, hipStream_t stream)
{
    const size_t pieces = static_cast<size_t>(p.m) * (p.pitch / 8);
    if (p.parts == 1 || pieces == 0) return DPEP_OK;
    join_kernel<kType, kFinish><<<static_cast<unsigned>((pieces + 255) / 256), 256, 0, stream>>>(p);
    return launch_status("product's parts");
}
template <int kType, bool kTransA, bool kTransB, Finish kFinish>
int launch(Product p, const Cut& c, void* partial, hipStream_t stream)
{
    if (p.m == 0 || p.columns == 0) return DPEP_OK;
    if constexpr (!kTransA && !kTransB) {
        if (c.way == kStream) {
            const Stream shape = stream_of(p.m, c.n_tiles);
            const dim3 grid((c.n_tiles + shape.groups - 1) / shape.groups, c.m_tiles);
            if (shape.blocks == 1 && shape.groups == 2) stream_kernel<kType, kFinish, 2, 1, 3><<<grid, kThreads, 0, stream>>>(p);
            else if (shape.blocks == 1 && shape.stages == 5) stream_kernel<kType, kFinish, 1, 1, 5><<<grid, kThreads, 0, stream>>>(p);
            else if (shape.blocks == 1) stream_kernel<kType, kFinish, 1, 1, 2><<<grid, kThreads, 0, stream>>>(p);
            else if (shape.blocks == 2 && shape.groups == 2) stream_kernel<kType, kFinish, 2, 2, 2><<<grid, kThreads, 0, stream>>>(p);
            else if (shape.blocks == 2) stream_kernel<kType, kFinish, 1, 2, 3><<<grid, kThreads, 0, stream>>>(p);
            else stream_kernel<kType, kFinish, 1, 4, 2><<<grid, kThreads, 0, stream>>>(p);
            return launch_status("product of few rows");
        }
    }
    p = cut_up(p, c, partial);
    const dim3 grid(static_cast<unsigned>(c.m_tiles) * c.n_tiles * c.parts);
    if (c.way == kLargeTiles) tile_kernel<kType, kTransA, kTransB, kFinish, kLargeTiles><<<grid, kThreads, 0, stream>>>(p);
    else if (c.way == kPairs) tile_kernel<kType, kTransA, kTransB, kFinish, kPairs><<<grid, kThreads, 0, stream>>>(p);
    else tile_kernel<kType, kTransA, kTransB, kFinish, kRing><<<grid, kThreads, 0, stream>>>(p);
    if (int rc = launch_status("product"); rc != DPEP_OK) return rc;
    return join<kType, kFinish>(p, stream);
}

// When `slots` that take tiles as they get free are done with the tiles of three products, tiles[i] of us[i] each, one product after the other.
double done_after(int slots, const long long (&tiles)[3], const double (&us)[3])
{
    double free_at[8] = {};  // groups of slots that get free together, at most one more for each product begun: the first group's rest and those moved on
    int slots_of[8] = {slots}, groups = 1;
    double end = 0;
    for (int i = 0; i < 3; ++i) {
        long long left = tiles[i];
        if (left == 0) continue;
        const long long rounds = std::max(0ll, left / slots - 2);  // (every slot takes these)
        for (int g = 0; g < groups; ++g) free_at[g] += static_cast<double>(rounds) * us[i];
        left -= rounds * slots;
        while (left > 0) {
            const int first = static_cast<int>(std::min_element(free_at, free_at + groups) - free_at);
            const int taken = static_cast<int>(std::min<long long>(left, slots_of[first]));
            const double then = free_at[first] + us[i];
            if (taken < slots_of[first]) {
                slots_of[first] -= taken;
                free_at[groups] = then;
                slots_of[groups++] = taken;
            } else {
                free_at[first] = then;
            }
            left -= taken;
        }
    }
    for (int g = 0; g < groups; ++g) end = std::max(end, free_at[g]);
    return end;
}

// Three products of 16-bit values without a part of another's operands: together in one launch, long tiles first and short ones to fill up, if that is quicker than one after
// the other with 4 us for a launch; a product of long k may be split there too.
// (8192 tokens, 4096 and 2048 values: 605 us with the product before them together in large tiles, 690 apart; 2048 tokens, 2048 and 1024: 72 in large tiles, 80 in pairs, 83 in the
// ring, 86 apart; 16000, 640 and 160: 127 in the ring, 69 apart, with k in parts; 6175, 912 and 240, both directions:
// 95 without parts, 75 with.)
struct Together {
    bool quicker = false;
    Way way = kRing;
    int order[3] = {0, 1, 2};
    Cut cuts[3] = {};  // of the products, by their own number
    size_t bytes = 0;  // of the parts' sums of all
};
Together together_of(const int (&m)[3], const int (&columns)[3], const int (&k)[3], const Cut (&apart)[3])
{
    Together best;
    double least = 8 + apart[0].us + apart[1].us + apart[2].us;
    for (const Way way : {kRing, kPairs, kLargeTiles})
        for (const int most : {1 << 30, 64, 32, 16, 8}) {  // steps of a part
            const int tile = way == kLargeTiles ? 256 : 128;
            Together now;
            now.way = way;
            double joins = 0;
            bool cut = false;
            for (int i = 0; i < 3; ++i) {
                Cut& c = now.cuts[i];
                const int steps = std::max(1, (k[i] * 2 + kStepBytes - 1) / kStepBytes), wanted = std::min(16, (steps - 1) / most + 1);
                c.m_tiles = (m[i] + tile - 1) / tile;
                c.n_tiles = (columns[i] + tile - 1) / tile;
                c.part_steps = (steps + wanted - 1) / wanted;
                c.parts = (steps + c.part_steps - 1) / c.part_steps;
                c.bytes = c.parts == 1 ? 0 : static_cast<size_t>(c.parts) * m[i] * ((columns[i] + 7) / 8 * 8) * 4;
                if (c.parts == 1 || m[i] == 0) continue;
                cut = true;
                joins += join_us(c.parts, c.bytes);
                now.bytes += c.bytes;
            }
            if (most != 1 << 30 && !cut) continue;
            std::sort(now.order, now.order + 3, [&](int x, int y) { return now.cuts[x].part_steps > now.cuts[y].part_steps; });
            long long tiles[3], all = 0;
            double us[3], bytes = static_cast<double>(now.bytes);
            for (int i = 0; i < 3; ++i) {
                const Cut& c = now.cuts[now.order[i]];
                tiles[i] = static_cast<long long>(c.m_tiles) * c.n_tiles * c.parts;
                us[i] = tile_us(way, c.part_steps);
                all += tiles[i];
                bytes += 2.0 * ((static_cast<double>(m[i]) + columns[i]) * k[i] + static_cast<double>(m[i]) * columns[i]);
            }
            const double done = joins + std::max(done_after(at_once(way), tiles, us) * (way == kPairs && all <= 256 ? 0.75 : 1.0), memory_us(way, all, bytes));
            if (all <= kMostWorkgroups && done < least) {
                least = done;
                best = now;
                best.quicker = true;
            }
        }
    return best;
}

template <int kType>
int launch_three(const Product (&products)[3], const Cut (&apart)[3], const Together& together, void* partial, hipStream_t stream)
{
    if (!together.quicker) {
        for (int i = 0; i < 3; ++i) {
            const int rc = products[i].turned_a != 0 ? launch<kType, true, true, kStore>(products[i], apart[i], partial, stream)
                                                     : launch<kType, false, true, kStore>(products[i], apart[i], partial, stream);
            if (rc != DPEP_OK) return rc;
        }
        return DPEP_OK;
    }
    Products all = {};
    uint8_t* sums = static_cast<uint8_t*>(partial);
    for (int i = 0; i < 3; ++i) {
        const Cut& c = together.cuts[together.order[i]];
        Product& p = all.of[i] = cut_up(products[together.order[i]], c, sums);
        sums += c.bytes;
        all.begin[i + 1] = all.begin[i] + static_cast<unsigned>(p.m_tiles) * p.n_tiles * p.parts;
    }
    if (together.way == kLargeTiles) products_kernel<kType, kLargeTiles><<<all.begin[3], kThreads, 0, stream>>>(all);
    else if (together.way == kPairs) products_kernel<kType, kPairs><<<all.begin[3], kThreads, 0, stream>>>(all);
    else products_kernel<kType, kRing><<<all.begin[3], kThreads, 0, stream>>>(all);
    if (int rc = launch_status("products"); rc != DPEP_OK) return rc;
    for (const Product& p : all.of)
        if (int rc = join<kType, kStore>(p, stream); rc != DPEP_OK) return rc;
    return DPEP_OK;
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

// How a block's products are cut up, and its scratch: the rows between the products, then the parts' sums of one product at a time.
struct ForwardCuts {
    Cut gate_up, down;
    size_t scratch;
    ForwardCuts(int tokens, int hidden, int inter)
        : gate_up(cut_of(tokens, inter, hidden * 2, true, false)),
          down(cut_of(tokens, hidden, inter * 2, false, false)),
          scratch(whole(static_cast<size_t>(tokens) * inter * 2) + std::max(gate_up.bytes, down.bytes))
    {
    }
};
struct BackwardCuts {
    Cut rows, three[3];  // dh; dx, dWgu, dWd, apart
    Together together;
    size_t scratch;
    BackwardCuts(int tokens, int hidden, int inter)
        : rows(cut_of(tokens, inter, hidden * 2, false, true)),
          three{cut_of(tokens, hidden, inter * 4, false, true), cut_of(2 * inter, hidden, tokens * 2, false, true), cut_of(hidden, inter, tokens * 2, false, true)},
          together(together_of({tokens, 2 * inter, hidden}, {hidden, hidden, inter}, {2 * inter, tokens, tokens}, three)),
          scratch(whole(static_cast<size_t>(tokens) * inter * 2) + whole(static_cast<size_t>(tokens) * inter * 4) +
                  std::max(rows.bytes, together.quicker ? together.bytes : std::max(three[0].bytes, std::max(three[1].bytes, three[2].bytes))))
    {
    }
};

// Sizes of a block that its entry points take.
inline bool block_fits(int tokens, int hidden, int inter)
{
    const auto dim = [](int d) { return d >= 8 && d % 8 == 0 && d <= DPEP_FFN_MAX_DIM; };
    return tokens >= 0 && tokens <= DPEP_FFN_MAX_TOKENS && dim(hidden) && dim(inter);
}
inline bool product_fits(int rows, int n, int k)
{
    return rows >= 0 && rows <= DPEP_W8_MAX_ROWS && n >= 1 && n <= DPEP_W8_MAX_N && k >= 16 && k % 16 == 0 && k <= DPEP_W8_MAX_K &&
           (rows + 255ll) / 256 * ((n + 255ll) / 256) <= kMostWorkgroups;
}
inline dpep_product_choice choice_of(const Cut& c, int m, bool together)
{
    dpep_product_choice choice = {c.way, c.parts, 0, 0, 0, together, static_cast<int64_t>(c.m_tiles) * c.n_tiles * c.parts};
    if (c.way != kStream) return choice;
    const Stream shape = stream_of(m, c.n_tiles);
    choice.stream_groups = shape.groups, choice.stream_blocks = shape.blocks, choice.stream_stages = shape.stages;
    choice.workgroups = static_cast<int64_t>((c.n_tiles + shape.groups - 1) / shape.groups) * c.m_tiles;
    return choice;
}

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
    return block_fits(num_tokens, hidden, inter) ? ForwardCuts(num_tokens, hidden, inter).scratch : 0;
}

int dpep_gated_ffn(const dpep_ffn* f, const void* x, int num_tokens, void* y, float* kept, void* scratch, void* stream)
{
    if (int rc = check_ffn(f, "gated_ffn", num_tokens); rc != DPEP_OK) return rc;
    if (num_tokens == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && y != nullptr && scratch != nullptr && aligned16(x) && aligned16(y) && aligned16(kept) && aligned16(scratch),
                 "gated_ffn: a NULL or misaligned buffer");
    const size_t rows = static_cast<size_t>(num_tokens) * f->hidden * 2, half = static_cast<size_t>(f->hidden) * f->inter * 2, products = static_cast<size_t>(num_tokens) * f->inter * 8;
    const ForwardCuts cuts(num_tokens, f->hidden, f->inter);
    const Span written[] = {{y, rows}, {kept, products}, {scratch, cuts.scratch}};
    const Span read[] = {{x, rows}, {f->gate_up, 2 * half}, {f->down, half}};
    DPEP_REQUIRE(apart(written, read), "gated_ffn: an output or scratch overlaps an input or one another");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    void* const partial = static_cast<uint8_t*>(scratch) + whole(static_cast<size_t>(num_tokens) * f->inter * 2);
    return by_type(f->type, [&](auto type) {
        constexpr int kType = decltype(type)::value;
        Product p = {x, f->gate_up, num_tokens, f->inter, f->hidden, {}};
        p.out.c = scratch;
        p.out.kept = kept;
        if (int rc = launch<kType, false, false, kGated>(p, cuts.gate_up, partial, s); rc != DPEP_OK) return rc;
        p = {scratch, f->down, num_tokens, f->hidden, f->inter, {}};
        p.out.c = y;
        return launch<kType, false, false, kStore>(p, cuts.down, partial, s);
    });
}

size_t dpep_gated_ffn_backward_scratch_bytes(int num_tokens, int hidden, int inter)
{
    return block_fits(num_tokens, hidden, inter) ? BackwardCuts(num_tokens, hidden, inter).scratch : 0;
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
    const Span read[] = {{grad_y, rows}, {x, rows}, {kept, products}, {f->gate_up, 2 * half}, {f->down, half}};
    const Span outputs[] = {{grad_x, rows}, {grad_gate_up, 2 * half}, {grad_down, half}};
    const BackwardCuts cuts(num_tokens, f->hidden, f->inter);
    const Span aside[] = {{scratch, cuts.scratch}};
    DPEP_REQUIRE(apart(outputs, {Span{nullptr, 0}}), "gated_ffn_backward: two outputs overlap");
    DPEP_REQUIRE(apart(outputs, read) && apart(aside, read) && apart(aside, outputs), "gated_ffn_backward: an output or scratch overlaps an input or one another");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    void* const h = scratch;
    void* const dz = static_cast<uint8_t*>(scratch) + whole(static_cast<size_t>(num_tokens) * f->inter * 2);
    void* const partial = static_cast<uint8_t*>(dz) + whole(static_cast<size_t>(num_tokens) * f->inter * 4);
    return by_type(f->type, [&](auto type) {
        constexpr int kType = decltype(type)::value;
        Product p = {grad_y, f->down, num_tokens, f->inter, f->hidden, {}};
        p.out.c = dz;
        p.out.kept = const_cast<float*>(kept);
        p.out.h = h;
        if (int rc = launch<kType, false, true, kGradient>(p, cuts.rows, partial, s); rc != DPEP_OK) return rc;
        Product products[3] = {{dz, f->gate_up, num_tokens, f->hidden, 2 * f->inter, {}},
                               {dz, x, 2 * f->inter, f->hidden, num_tokens, {}},
                               {grad_y, h, f->hidden, f->inter, num_tokens, {}}};
        products[0].out.c = grad_x;
        products[1].out.c = grad_gate_up;
        products[2].out.c = grad_down;
        products[1].turned_a = products[2].turned_a = 1;
        return launch_three<kType>(products, cuts.three, cuts.together, partial, s);
    });
}

int dpep_product_choices(int operation, int rows, int a, int b, dpep_product_choice* choices)
{
    DPEP_REQUIRE(choices != nullptr, "product_choices: choices is NULL");
    DPEP_REQUIRE(operation >= DPEP_PRODUCTS_FFN && operation <= DPEP_PRODUCTS_W8, "product_choices: operation=%d is not one of DPEP_PRODUCTS_*", operation);
    DPEP_REQUIRE(operation == DPEP_PRODUCTS_W8 ? product_fits(rows, a, b) : block_fits(rows, a, b), "product_choices: %d, %d and %d are not taken", rows, a, b);
    if (operation == DPEP_PRODUCTS_W8) {
        choices[0] = choice_of(cut_of(rows, a, b, false, false), rows, false);
        return 1;
    }
    if (operation == DPEP_PRODUCTS_FFN) {
        const ForwardCuts cuts(rows, a, b);
        choices[0] = choice_of(cuts.gate_up, rows, false);
        choices[1] = choice_of(cuts.down, rows, false);
        return 2;
    }
    const BackwardCuts cuts(rows, a, b);
    choices[0] = choice_of(cuts.rows, rows, false);
    for (int i = 0; i < 3; ++i) {
        choices[1 + i] = choice_of(cuts.together.quicker ? cuts.together.cuts[i] : cuts.three[i], rows, cuts.together.quicker);
        if (cuts.together.quicker) choices[1 + i].way = cuts.together.way;
    }
    return 4;
}

size_t dpep_w8_matmul_scratch_bytes(int num_rows, int n, int k)
{
    return product_fits(num_rows, n, k) ? cut_of(num_rows, n, k, false, false).bytes : 0;
}

int dpep_w8_matmul(const dpep_w8* w, const int8_t* x, const float* x_scales, int num_rows, int type, void* y, void* scratch, void* stream)
{
    DPEP_REQUIRE(w != nullptr, "w8_matmul: weights is NULL");
    DPEP_REQUIRE(type == DPEP_TYPE_F32 || type == DPEP_TYPE_BF16 || type == DPEP_TYPE_F16, "w8_matmul: type=%d is not one of DPEP_TYPE_*", type);
    DPEP_REQUIRE(w->k >= 16 && w->k % 16 == 0 && w->k <= DPEP_W8_MAX_K, "w8_matmul: K=%d is not a multiple of 16 in [16, %d]", w->k, DPEP_W8_MAX_K);
    DPEP_REQUIRE(w->n >= 1 && w->n <= DPEP_W8_MAX_N, "w8_matmul: N=%d is not in [1, %d]", w->n, DPEP_W8_MAX_N);
    DPEP_REQUIRE(num_rows >= 0 && num_rows <= DPEP_W8_MAX_ROWS, "w8_matmul: T=%d is not in [0, %d]", num_rows, DPEP_W8_MAX_ROWS);
    DPEP_REQUIRE(product_fits(num_rows, w->n, w->k), "w8_matmul: T=%d times N=%d is too large", num_rows, w->n);
    DPEP_REQUIRE(w->codes != nullptr && w->scales != nullptr && aligned16(w->codes), "w8_matmul: a NULL or misaligned matrix");
    if (num_rows == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && x_scales != nullptr && y != nullptr && aligned16(x), "w8_matmul: a NULL or misaligned buffer");
    const Cut cut = cut_of(num_rows, w->n, w->k, false, false);
    DPEP_REQUIRE(cut.bytes == 0 || (scratch != nullptr && aligned16(scratch)), "w8_matmul: scratch is NULL or misaligned");
    const size_t results = static_cast<size_t>(num_rows) * w->n * (type == DPEP_TYPE_F32 ? 4 : 2);
    const Span written[] = {{y, results}, {scratch, cut.bytes}};
    const Span read[] = {{x, static_cast<size_t>(num_rows) * w->k}, {x_scales, num_rows * 4ull}, {w->codes, static_cast<size_t>(w->n) * w->k}, {w->scales, w->n * 4ull}};
    DPEP_REQUIRE(apart(written, read), "w8_matmul: y or scratch overlaps an input or one another");
    Product p = {x, w->codes, num_rows, w->n, w->k, {}};
    p.out.c = y;
    p.out.row_scale = x_scales;
    p.out.column_scale = w->scales;
    p.out.type = type;
    return launch<kInt8, false, false, kScaled>(p, cut, scratch, static_cast<hipStream_t>(stream));
}

}  // extern "C"
