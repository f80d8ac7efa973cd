// Products of a few rows with matrices held in 4 bits with group scales: one matrix, and the experts of a routed layer.
//
//   W[n,k] = (q[n,k] - zero[n,k/G]) * scale[n,k/G],  y[m,n] = sum_k x[m,k] W[n,k]
//   experts: h = silu(W1g[e] x_t) * (W1u[e] x_t),  y_t = sum_s w_ts W2[e] h
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.h"

#pragma clang fp contract(off)

namespace dpep {
namespace {

constexpr int kMaxRoutes = DPEP_W4_MAX_ROUTES;
constexpr int kMaxK = DPEP_W4_MAX_K;

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

// The products run on the matrix cores (16 x 16 x 32): rows of x against 16 rows of W, whose codes become numbers without arithmetic: a
// code's bits under the exponent of 16 are the 16-bit number 16 + q.  Over a group, with X = sum of x,
//   sum x W = scale (sum x (16 + q) - (16 + zero) X)
// where the accumulator starts at -(16 + zero) X, so a group ends with one multiply-add for every result.
//
// A wave streams pairs of 16-byte loads that cover 8 rows of whole 128-byte lines each (16 rows x 256 of k, a "unit"), which HBM serves as fast
// as contiguous kilobytes (6.9 TB/s; 16 rows of 64 bytes: 5.5).  Lane l loads row l % 8 of each half, chunk (32 values) l / 16 + 4 (l / 8 % 2); swapping
// between lanes 8 apart makes of the two loads the two operands X and Y, in which lane l holds row l % 16 and chunk l / 16 of the
// unit's first and second 128 values.
//
// An MFMA adds up the four chunks of its operand.  Where a group is shorter than 128 values these belong to kDiag = 2 or 4 groups: the rows of the
// other operand are then (group, token) with zeros outside the row's own group, so that every group has accumulators of its own, at 16 / kDiag
// tokens an MFMA; in all cases a lane's results belong to the group of the chunk that the lane loaded.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / kWave, kLogWaves = 3;
constexpr int kUnit = 256;  // values of k

enum Kind { kMatvec, kGateUp, kDown };

// One launch's matrices and how they are walked.
struct Product {
    const uint8_t* packed;
    const uint16_t* scales;
    const uint8_t* zeros;
    int n, k, group;    // of one matrix
    int units, groups;  // of a row
    int group_inverse;  // ceil(2^20 / (group / 128)), for groups of 128 and more
    bool ragged;        // units and groups do not end together: a unit's scales may reach past their row
    size_t all_scales;  // of all matrices
    int split, log_split;  // waves that share a tile's k
    int tile_groups;    // of a matrix, kTiles tiles each
    int steps;          // a matrix in steps of a workgroup: kWaves / split tile groups at a time
    int batch;          // steps whose results wait in LDS for one another
    int row_cap;        // rows of x held in LDS
    // rows: matvec: x [rows, k]; gate_up: x [token, k]; down: the routes' (high, low) rows [route][2][k]
    const uint16_t* x;
    int rows;
    Ids ids;
    int routes, topk;
    const float* route_weights;
    void* out;  // matvec: y; gate_up: the down product's x; down: [route][n] fp32
};

// The constants that make numbers of codes, in registers (an instruction that masks and inserts takes no literals).
template <bool kHalf>
struct Codes {
    uint32_t mask, sixteen;
    __device__ __forceinline__ Codes()
    {
        asm("s_mov_b32 %0, %1" : "=s"(mask) : "i"(kHalf ? 0x03C003C0u : 0x00780078u));
        asm("v_mov_b32 %0, %1" : "=v"(sixteen) : "i"(kHalf ? 0x4C004C00u : 0x41804180u));
    }
    // Eight codes, values (0, 4), (1, 5), (2, 6) and (3, 7), each 16 + q.
    __device__ __forceinline__ u32x4 unpack(uint32_t w) const
    {
        if constexpr (kHalf) return u32x4{((w << 6) & mask) | sixteen, ((w << 2) & mask) | sixteen, ((w >> 2) & mask) | sixteen, ((w >> 6) & mask) | sixteen};
        return u32x4{((w << 3) & mask) | sixteen, ((w >> 1) & mask) | sixteen, ((w >> 5) & mask) | sixteen, ((w >> 9) & mask) | sixteen};
    }
};
template <bool kHalf>
__device__ __forceinline__ f32x4 multiply(u32x4 x, u32x4 w, f32x4 c)
{
    if constexpr (kHalf) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, w), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w), c, 0, 0, 0);
}

// Waits for LDS alone: the loads in flight stay in flight.
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A launch's LDS: the rows in the MFMA's order, their groups' sums, the waves' results, what is kept of the routes.  Rows come in fours (the rows of
// one lane's results); what lies behind the last is read and not used.
struct LdsPlan {
    int sums, results, counts, routes, weights, bytes;
    int lanes;  // of a wave that hold results of these rows
    __host__ __device__ LdsPlan(int units, int diag, int blocks, int tiles, int rows, int batch, int experts, int num_routes, bool weighted)
    {
        const int fours = (rows + 3) / 4, tokens = 16 / diag;
        lanes = diag == 1 && blocks == 1 ? fours * 16 : kWave;
        sums = (units * 32 * rows + tokens * blocks) * 16;
        results = sums + units * 2 * diag * fours * 16 + tokens * blocks * 4;
        counts = results + batch * kWaves * tiles * blocks * 4 * lanes * 4;
        routes = counts + (experts + 63) / 64 * 256;
        weights = routes + (num_routes + 3) / 4 * 16;  // (an expert each, and a list of those of one expert)
        bytes = weights + (weighted ? (num_routes + 3) / 4 * 16 : 0);
    }
};

// A workgroup takes an even share of all steps: of the matrices that have rows one after the other (matvec: of the passes over the rows), each
// with the rows it multiplies in LDS.
//
// Few rows: reading the codes bounds it.  Sixteen tokens through 8 of 256 experts, 2.0 GB of weights: 351 to 367 us in all, 5.5 to 5.7 TB/s.  One token, 121 MB and
// 60 MB: 27 and 18 us, 4.4 and 3.3 TB/s, of which 5 to 6 pass before the first weights are asked for (ids, then rows, then the barrier) and 2
// behind the last.  Many rows: the rows' way into LDS, once for every 16 columns and pass (64 rows through 4096 x 7168: 42 us).
// The experts' products with zero points and one block keep two to seven registers a lane on the stack (two workgroups to a CU leave 128);
// with four blocks they have a CU to themselves, and 161 to 168 registers.
template <Kind kKind, bool kHalf, bool kZeros, int kDiag, int kBlocks, bool kStreamed>
__global__ __launch_bounds__(kThreads, kBlocks == 1 ? 4 : 2) void product_kernel(const Product p)
{
    constexpr bool kHalfRows = kHalf && kKind != kDown;  // the down product's rows are BF16 pairs whatever the type
    constexpr int kTiles = kKind == kMatvec ? 1 : 2;     // tiles of 16 rows of W to a tile group; gate_up: a gate tile and its up tile
    // Units in flight.  The waves of a CU (sixteen, 4 KiB each) need not ask for more: with two units each, requests queued for 5 us, and so did
    // everything that was cold, instructions among it (one token through 8 of 256 experts 65 us against 51, sixteen tokens 370 against 350).
    constexpr int kAhead = kKind == kMatvec ? 2 : 1;
    constexpr int kTokens = 16 / kDiag;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ __attribute__((aligned(16))) uint32_t zero16[4];
    const int experts = kKind == kMatvec ? 0 : p.ids.local;
    const LdsPlan plan(p.units, kDiag, kBlocks, kTiles, p.row_cap, p.batch, experts, p.routes, kKind == kGateUp);
    unsigned char* const x_lds = lds;
    float* const sums_lds = reinterpret_cast<float*>(lds + plan.sums);
    float* const results = reinterpret_cast<float*>(lds + plan.results);  // [wave][tile][block][four of a lane][lane]
    int* const counts = reinterpret_cast<int*>(lds + plan.counts);
    int16_t* const expert_of = reinterpret_cast<int16_t*>(lds + plan.routes);
    uint16_t* const my_routes = reinterpret_cast<uint16_t*>(expert_of) + p.routes;
    float* const route_weights = reinterpret_cast<float*>(lds + plan.weights);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, chunk = lane >> 4;
    if (tid < 4) zero16[tid] = 0;
    // Passes of row_cap rows: matvec's, or each expert's; lane l counts those of experts l * per_lane and on.
    const int per_lane = (experts + kWave - 1) / kWave;
    int passes = 0, passes_before = 0, matrices = 0;
    if constexpr (kKind == kMatvec) {
        matrices = (p.rows + p.row_cap - 1) / p.row_cap;
    } else {
        for (int e = tid; e < per_lane * kWave; e += kThreads) counts[e] = 0;
        __syncthreads();
        for (int i = tid; i < p.routes; i += kThreads) {
            const int e = p.ids[i];
            if constexpr (kKind == kGateUp) route_weights[i] = p.route_weights[i];
            expert_of[i] = static_cast<int16_t>(e);
            if (e >= 0) atomicAdd(&counts[e], kKind == kDown ? 2 : 1);
        }
        __syncthreads();
        for (int i = 0; i < per_lane; ++i) passes += (counts[lane * per_lane + i] + p.row_cap - 1) / p.row_cap;
        const int until = wave_scan(passes);
        passes_before = until - passes;
        matrices = __builtin_amdgcn_readlane(until, 63);
    }
    const int all_steps = matrices * p.steps;
    const int even = all_steps / static_cast<int>(gridDim.x), over = all_steps - even * static_cast<int>(gridDim.x), block = blockIdx.x;
    int step = block * even + min(block, over);
    const int end_step = step + even + (block < over ? 1 : 0);

    // What this wave streams: units first_unit .. last_unit - 1 of its tile groups.
    const int split = p.split, lanes_of_groups = kWaves / split;
    const int mine = wave >> p.log_split;
    // (shares of k differ by a unit where the split leaves a rest, so the waves take them in turn)
    auto first_unit = [&](int step) { return p.units * ((wave + step) & (split - 1)) >> p.log_split; };
    auto last_unit = [&](int step) { return p.units * (((wave + step) & (split - 1)) + 1) >> p.log_split; };
    const int slots = ((p.units + split - 1) / split + 3) / 4 * 4;  // to a step, the same for all waves
    const int matrix_rows = kKind == kGateUp ? p.n / 2 : p.n;  // among which tiles are counted
    const int half_k = p.k / 2;
    // (a matrix of fewer than 16 rows: lanes past its end load its last row; the last tile of others is moved up to end with the matrix)
    const int loaded_chunk = chunk + 4 * ((lane >> 3) & 1);
    const uint32_t row_low = min(lane & 7, matrix_rows - 1) * half_k, row_high = min((lane & 7) + 8, matrix_rows - 1) * half_k;
    const int tail_chunk = (p.units - 1) * 8 + loaded_chunk < p.k / 32 ? loaded_chunk : 0;  // chunks behind k: any that exist (x is zero there)
    const uint32_t scale_row = min(col, matrix_rows - 1) * p.groups;
    auto tile_row = [&](int g, int tile) {  // of the matrix: first row of one of a tile group's tiles
        g = min(g, p.tile_groups - 1);
        if constexpr (kKind == kGateUp) return min(g * 16, max(matrix_rows - 16, 0)) + tile * matrix_rows;
        return min((g * kTiles + tile) * 16, max(matrix_rows - 16, 0));
    };
    const Codes<kHalfRows> codes;
    // Where a lane reads x: token lane % 16 (of its group's rows), chunk lane / 16; zeros outside the row's own group.
    const bool own = kDiag == 1 || chunk / (4 / kDiag) == col / kTokens;

    while (step < end_step) {
        const int matrix = step / p.steps, first_step = step - matrix * p.steps, steps = min(p.steps - first_step, end_step - step);
        step += steps;
        int expert = 0, count = p.rows, first_row = matrix * p.row_cap;
        if constexpr (kKind != kMatvec) {
            // The expert of the matrix-th pass, and which of its passes that is.
            const int at = __ffsll(__ballot(matrix >= passes_before && matrix < passes_before + passes)) - 1;
            int skip = matrix - __builtin_amdgcn_readlane(passes_before, at);
            expert = at * per_lane;
            for (;; ++expert) {
                count = __builtin_amdgcn_readfirstlane(counts[expert]);
                const int here = (count + p.row_cap - 1) / p.row_cap;
                if (skip < here) break;
                skip -= here;
            }
            first_row = skip * p.row_cap;
        }
        const uint8_t* const packed = p.packed + static_cast<size_t>(expert) * p.n * half_k;
        const uint16_t* const scales = p.scales + static_cast<size_t>(expert) * p.n * p.groups;
        const uint8_t* const zeros = kZeros ? p.zeros + static_cast<size_t>(expert) * p.n * p.groups : nullptr;

        struct Slot {
            u32x4 low[kTiles], high[kTiles];
        };
        // (real = false: a slot that nobody consumes, filled all the same from one place, so that the loads in flight can be counted)
        auto load = [&](Slot& s, int g, int u, bool real) {
            asm volatile("" : "+s"(u));  // (as below)
            const uint32_t at = (u == p.units - 1 ? tail_chunk : loaded_chunk) * 16;
            const uint32_t low = real ? row_low + at : 0, high = real ? row_high + at : 0;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int row = tile_row(g, t);
                const uint8_t* const base = packed + static_cast<size_t>(row) * half_k + u * (kUnit / 2);
                if constexpr (kStreamed) {
                    s.low[t] = load16_nt(base + low);
                    s.high[t] = load16_nt(base + high);
                } else {
                    s.low[t] = load16(base + low);
                    s.high[t] = load16(base + high);
                }
            }
        };

        // Scales: a lane takes those of row l % 16 and of the (l / 16)-th of four units, 2 kDiag of them next to one another, in one load.  (One load for a
        // unit and a lane's own two would touch 16 lines for 64 bytes each time; these filled the queue of misses: 443 us for the
        // largest call, 388 with this and results of several steps behind one barrier.)
        struct Scales {
            uint32_t scale[kTiles][kDiag], zero[kTiles][kDiag == 4 ? 2 : 1];
        };
        auto first_scale = [&](int unit) { return kDiag == 1 ? (2 * unit * p.group_inverse) >> 20 : unit * 2 * kDiag; };  // of a unit, in its row
        auto scales_left = [&](int row) {  // from the beginning of a row to the end of the tensor
            const size_t left = p.all_scales - (static_cast<size_t>(expert) * p.n + row) * p.groups;
            return static_cast<int>(left < (1u << 30) ? left : 1u << 30);
        };
        auto block_unit = [&](int step, int block) { return min(first_unit(step) + block * 4 + chunk, last_unit(step) - 1); };
        auto load_scales = [&](Scales& s, int step, int block) {
            const uint32_t at = scale_row + first_scale(block_unit(step, block));
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int row = tile_row(step * lanes_of_groups + mine, t);
                const size_t begin = static_cast<size_t>(row) * p.groups;
                const uint8_t* const scale = reinterpret_cast<const uint8_t*>(scales + begin);
                if (p.ragged && p.all_scales < 2 * kDiag) {  // fewer than one load takes: one by one
                    for (int d = 0; d < kDiag; ++d) s.scale[t][d] = 0;
                    if constexpr (kZeros) s.zero[t][0] = s.zero[t][kDiag == 4 ? 1 : 0] = 0;
                    const int left = scales_left(row) - static_cast<int>(at);
#pragma unroll
                    for (int i = 0; i < 2 * kDiag; ++i)  // (indices that are constants keep these arrays in registers)
                        if (i < left) {
                            s.scale[t][i / 2] |= static_cast<uint32_t>((scales + begin)[at + i]) << (16 * (i % 2));
                            if constexpr (kZeros) s.zero[t][i / 4] |= static_cast<uint32_t>((zeros + begin)[at + i]) << (8 * (i % 4));
                        }
                    continue;
                }
                const uint32_t from = p.ragged ? min(at, static_cast<uint32_t>(scales_left(row) - 2 * kDiag)) : at;
                __builtin_memcpy(s.scale[t], scale + 2 * from, 4 * kDiag);
                if constexpr (kZeros) __builtin_memcpy(s.zero[t], zeros + begin + from, 2 * kDiag);
            }
        };
        // What becomes of them: for each of the four units a register with a lane's two scales (zero points), those of operand X below those of Y.
        auto spread = [&](uint32_t (&pairs)[kDiag], uint32_t (&of_unit)[4], int step, int block, int t) {
            if (p.ragged) {
                // a load that was moved back to end with the tensor is shifted, and what lies behind the row becomes zero
                const int unit = block_unit(step, block), start = first_scale(unit), row = tile_row(step * lanes_of_groups + mine, t);
                const int over = p.all_scales < 2 * kDiag ? 0 : max(0, static_cast<int>(scale_row) + start + 2 * kDiag - scales_left(row));
                if constexpr (kDiag == 4) {
                    const bool four = (over & 4) != 0;
                    pairs[0] = four ? pairs[2] : pairs[0];
                    pairs[1] = four ? pairs[3] : pairs[1];
                }
                if constexpr (kDiag >= 2)
#pragma unroll
                    for (int d = 0; d < kDiag; ++d) pairs[d] = (over & 2) == 0 ? pairs[d] : d + 1 < kDiag ? pairs[d + 1] : 0u;
#pragma unroll
                for (int d = 0; d < kDiag; ++d) pairs[d] = (over & 1) == 0 ? pairs[d] : (pairs[d] >> 16) | (d + 1 < kDiag ? pairs[d + 1] << 16 : 0u);
                if constexpr (kDiag == 1) {  // long groups: both halves of a unit may be of one
                    const int second = ((2 * unit + 1) * p.group_inverse) >> 20;
                    if (second == start) pairs[0] = (pairs[0] & 0xffffu) | (pairs[0] << 16);
                    else if (second >= p.groups) pairs[0] &= 0xffffu;
                } else {
                    const int valid = p.groups - start;
#pragma unroll
                    for (int d = 0; d < kDiag; ++d) pairs[d] = 2 * d + 1 < valid ? pairs[d] : 2 * d < valid ? pairs[d] & 0xffffu : 0u;
                }
            }
            uint32_t both[kDiag];  // X and Y of the lane group
            if constexpr (kDiag == 1) both[0] = pairs[0];
            else
#pragma unroll
                for (int d = 0; d < kDiag / 2; ++d) {
                    both[2 * d] = (pairs[d] & 0xffffu) | (pairs[kDiag / 2 + d] << 16);
                    both[2 * d + 1] = (pairs[d] >> 16) | (pairs[kDiag / 2 + d] & 0xffff0000u);
                }
            // Rows of 16 lanes change places with registers, so that every lane has its own group's of all four units.
            auto swap16 = [](uint32_t& a, uint32_t& b) {  // odd rows of a with even rows of b
                const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
                a = r[0];
                b = r[1];
            };
            auto swap32 = [](uint32_t& a, uint32_t& b) {  // the upper half of a with the lower half of b
                const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
                a = r[0];
                b = r[1];
            };
            if constexpr (kDiag == 1) {
                of_unit[0] = of_unit[1] = both[0];
                swap16(of_unit[0], of_unit[1]);  // rows 0 0 2 2 and 1 1 3 3
                of_unit[2] = of_unit[0];
                of_unit[3] = of_unit[1];
                swap32(of_unit[0], of_unit[2]);
                swap32(of_unit[1], of_unit[3]);
            } else if constexpr (kDiag == 2) {
                of_unit[0] = both[0];
                of_unit[2] = both[1];
                swap32(of_unit[0], of_unit[2]);
                of_unit[1] = of_unit[0];
                of_unit[3] = of_unit[2];
                swap16(of_unit[0], of_unit[1]);
                swap16(of_unit[2], of_unit[3]);
            } else {
                of_unit[0] = both[0];
                of_unit[1] = both[1];
                of_unit[2] = both[2];
                of_unit[3] = both[3];
                swap16(of_unit[0], of_unit[1]);
                swap16(of_unit[2], of_unit[3]);
                swap32(of_unit[0], of_unit[2]);
                swap32(of_unit[1], of_unit[3]);
            }
        };

        lds_barrier();  // nobody reads the rows and routes that were there
        if constexpr (kKind != kMatvec) {  // (every wave makes the same list, and need not wait for another)
            int held = 0;
            for (int base = 0; base < p.routes; base += kWave) {
                const bool hit = base + lane < p.routes && expert_of[base + lane] == expert;
                const unsigned long long mask = __ballot(hit);
                if (hit) my_routes[held + __popcll(mask & ((1ull << lane) - 1))] = static_cast<uint16_t>(base + lane);
                held += __popcll(mask);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        const int rows = min(count - first_row, p.row_cap), padded = (rows + 3) & ~3;

        // Rows into LDS, an octet of values to a thread and turn, as the MFMA wants them: [unit][half][octet][chunk][row], an octet's pairs four apart.
        // Sixteen lanes next to one another have 128 values, so their groups' sums are a few exchanges away.  The weights are asked for when the
        // rows are there: behind weights in the CU's queue rows take 5 us to come, and the waves hold units that wait for them.
        const int pieces = rows * p.units * 32, per_row = p.units * 32;  // (units are whole: a multiple of 16)
        constexpr int kTurns = 2;
        u32x4 octets[kTurns];
        auto fetch = [&](int first) {
#pragma unroll
            for (int turn = 0; turn < kTurns; ++turn) {
                const int i = first + turn * kThreads, m = i / per_row, at = i - m * per_row, which = first_row + min(m, rows - 1);
                const uint16_t* from;
                if constexpr (kKind == kMatvec) from = p.x + static_cast<size_t>(which) * p.k;
                else if constexpr (kKind == kGateUp) from = p.x + static_cast<size_t>(my_routes[which] / p.topk) * p.k;
                else from = p.x + (static_cast<size_t>(my_routes[which >> 1]) * 2 + (which & 1)) * p.k;
                octets[turn] = load16(from + (at * 8 < p.k ? at * 8 : 0));
            }
        };
        auto put = [&](int first) {
#pragma unroll
            for (int turn = 0; turn < kTurns; ++turn) {
                const int i = first + turn * kThreads, m = i / per_row, at = i - m * per_row, c32 = at >> 2;
                if (i >= pieces) break;  // (sixteen lanes at a time)
                const u32x4 v = at * 8 < p.k ? octets[turn] : u32x4{0u, 0u, 0u, 0u};
                float sum = 0.0f;
#pragma unroll
                for (int d = 0; d < 4; ++d) sum += widen(v[d] & 0xffffu, kHalfRows) + widen(v[d] >> 16, kHalfRows);
                const u32x4 pairs = {(v[0] & 0xffffu) | (v[2] << 16), (v[0] >> 16) | (v[2] & 0xffff0000u), (v[1] & 0xffffu) | (v[3] << 16),
                                     (v[1] >> 16) | (v[3] & 0xffff0000u)};
                *reinterpret_cast<u32x4*>(x_lds + static_cast<size_t>((((c32 >> 2) * 4 + (at & 3)) * 4 + (c32 & 3)) * rows + m) * 16) = pairs;
                auto exchange = [&](auto control) {
                    sum += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(sum), control(), 0xf, 0xf, false));
                };
                exchange(std::integral_constant<int, 0xB1>{});                                // lane ^ 1
                exchange(std::integral_constant<int, 0x4E>{});                                // lane ^ 2: a chunk
                if constexpr (kDiag < 4) exchange(std::integral_constant<int, 0x141>{});  // the other chunk of two
                if constexpr (kDiag < 2) exchange(std::integral_constant<int, 0x140>{});  // the other two of four
                if ((at & (16 / kDiag - 1)) == 0) sums_lds[static_cast<size_t>(at / (16 / kDiag)) * padded + m] = kZeros ? -sum : -24.0f * sum;
            }
        };
        fetch(tid);

        Slot ring[kAhead];
        Scales next_scales;
        int load_step = first_step, load_slot = 0;
        auto load_next = [&](Slot& s) {
            const int u = first_unit(load_step) + load_slot, end = last_unit(load_step);
            load(s, load_step * lanes_of_groups + mine, min(u, end - 1), u < end);
            if (++load_slot == slots) {
                load_slot = 0;
                load_step = min(load_step + 1, first_step + steps - 1);
            }
        };
        put(tid);
        for (int i = tid + kTurns * kThreads; i < pieces; i += kTurns * kThreads) {
            fetch(i);
            put(i);
        }
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
        load_scales(next_scales, first_step, 0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load_next(ring[i]);

        f32x4 acc[kTiles][kBlocks] = {};
        const int x_lane = own ? (chunk * rows + min(col % kTokens, rows - 1)) * 16 : 0;
        auto consume = [&](const Slot& s, int u, const uint32_t (&scale_pair)[kTiles], const uint32_t (&zero_pair)[kTiles], int zero_byte) {
            asm volatile("" : "+s"(u));  // (or each of its LDS addresses becomes an induction variable in a register)
            // What LDS holds is asked for before the weights are waited for.
            auto x_at = [&](int part, int j) {
                return own ? x_lds + (part * 4 + j) * 4 * rows * 16 + x_lane : reinterpret_cast<const unsigned char*>(zero16);
            };
            u32x4 x[2][4];
            if constexpr (kBlocks == 1) {
#pragma unroll
                for (int f = 0; f < 2; ++f)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[f][j] = *reinterpret_cast<const u32x4*>(x_at(u * 2 + f, j));
                __builtin_amdgcn_sched_barrier(0);
            }
            u32x4 w[2][kTiles];
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    w[0][t][d] = __builtin_amdgcn_update_dpp(s.low[t][d], s.high[t][d], 0x128, 0xf, 0xc, false);
                    w[1][t][d] = __builtin_amdgcn_update_dpp(s.high[t][d], s.low[t][d], 0x128, 0xf, 0x3, false);
                }
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int part = u * 2 + f;
                f32x4 c[kTiles][kBlocks];
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    const int sub = kDiag == 1 ? 0 : chunk / (4 / kDiag), token = (kDiag == 1 ? chunk * 4 : kDiag == 2 ? (chunk & 1) * 4 : 0) + b * kTokens;
                    const f32x4 start = *reinterpret_cast<const f32x4*>(sums_lds + static_cast<size_t>(part * kDiag + sub) * padded + token);
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        c[t][b] = start;
                        if constexpr (kZeros) {
                            const float zero = 16.0f + static_cast<float>((zero_pair[t] >> (16 * f + 8 * zero_byte)) & 0xffu);
#pragma unroll
                            for (int i = 0; i < 4; ++i) c[t][b][i] *= zero;
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u32x4 q[kTiles];
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) q[t] = codes.unpack(w[f][t][j]);
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        u32x4 a;
                        if constexpr (kBlocks == 1) a = x[f][j];
                        else a = *reinterpret_cast<const u32x4*>(x_at(part, j) + (own ? b * kTokens * 16 : 0));
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) c[t][b] = multiply<kHalfRows>(a, q[t], c[t][b]);
                    }
                }
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    const float scale = widen(f == 0 ? scale_pair[t] & 0xffffu : scale_pair[t] >> 16, kHalf);
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][b][i] = fmaf(scale, c[t][b][i], acc[t][b][i]);
                }
                if constexpr (kBlocks > 1) __builtin_amdgcn_sched_barrier(0);  // (the other half's operands would be fetched here, and cost registers)
            }
        };

        // Results: the waves that share a tile leave theirs in LDS, those of a batch of steps behind one another; then as many lanes next to one
        // another add them up (for short groups also over the lanes that hold a tile's groups).
        const int step_results = kWaves * kTiles * kBlocks * 4 * plan.lanes;
        auto leave = [&](int place) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (lane < plan.lanes) results[place * step_results + (((wave * kTiles + t) * kBlocks + b) * 4 + i) * plan.lanes + lane] = acc[t][b][i];
                        acc[t][b][i] = 0.0f;
                    }
        };
        auto finish = [&](int from_step, int number) {
            lds_barrier();
            auto shared = [&](int place, int group, int tile, int m, int n, int w) {
                const int b = m / kTokens, token = m % kTokens;
                float sum = 0.0f;
#pragma unroll
                for (int d = 0; d < kDiag; ++d) {
                    const int from = kDiag == 1 ? token / 4 : kDiag == 2 ? token / 4 + 2 * d : d;
                    sum += results[place * step_results + ((((group * split + w) * kTiles + tile) * kBlocks + b) * 4 + token % 4) * plan.lanes + from * 16 + n];
                }
                if (split >= 2) sum += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(sum), 0xB1, 0xf, 0xf, false));   // lane ^ 1
                if (split >= 4) sum += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(sum), 0x4E, 0xf, 0xf, false));   // lane ^ 2
                if (split >= 8) sum += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(sum), 0x141, 0xf, 0xf, false));  // 7 - lane
                return sum;
            };
            constexpr int kOut = kKind == kGateUp ? 1 : kTiles;  // result tiles of a tile group
            const int per_step = lanes_of_groups * kOut * 16 * (kKind == kDown ? rows / 2 : rows) * split;
            for (int i = tid; i < per_step * number; i += kThreads) {  // (per_step is a multiple of 16: lanes that add up stay together)
                const int place = number == 1 ? 0 : i / per_step, at = i - place * per_step;
                const int w = at & (split - 1), o = at >> p.log_split, n = o & 15, tile = (o >> 4) % kOut, rest = (o >> 4) / kOut;
                const int group = rest & (lanes_of_groups - 1), m = rest >> (kLogWaves - p.log_split);
                const int g = (from_step + place) * lanes_of_groups + group;
                const int to = tile_row(g, tile) + n;
                const bool mine_to_store = w == 0 && g < p.tile_groups && to < matrix_rows;
                if constexpr (kKind == kMatvec) {
                    // A last tile that was moved up stores its own columns alone: it adds the shares of k in another order than the tile in front (they
                    // go round with the step), so the columns that both hold may differ in their last bits.  (Experts' matrices have whole tiles.)
                    const float y = shared(place, group, tile, m, n, w);
                    if (mine_to_store && to >= g * 16) static_cast<uint16_t*>(p.out)[static_cast<size_t>(first_row + m) * p.n + to] = narrow(y, kHalf);
                } else if constexpr (kKind == kGateUp) {
                    const float gate = shared(place, group, 0, m, n, w), up = shared(place, group, 1, m, n, w);
                    const int route = my_routes[first_row + m];
                    // The route's weight is folded in here.  Two BF16 numbers hold the product's high and low part, together 16 bits of mantissa.
                    const float h = gate / (1.0f + expf(-gate)) * up * route_weights[route];
                    const uint32_t high = f32_to_bf16(h);
                    uint16_t* const row = static_cast<uint16_t*>(p.out) + static_cast<size_t>(route) * 2 * matrix_rows + to;
                    if (mine_to_store) {
                        row[0] = static_cast<uint16_t>(high);
                        row[matrix_rows] = static_cast<uint16_t>(f32_to_bf16(h - bf16_to_f32(high)));
                    }
                } else {
                    const int route = my_routes[(first_row >> 1) + m];
                    const float y = shared(place, group, tile, 2 * m, n, w) + shared(place, group, tile, 2 * m + 1, n, w);
                    if (mine_to_store) static_cast<float*>(p.out)[static_cast<size_t>(route) * p.n + to] = y;
                }
            }
        };

        for (int done = 0; done < steps; done += p.batch) {
            const int number = min(p.batch, steps - done);
            for (int i = 0; i < number; ++i) {
                const int at_step = first_step + done + i, from = first_unit(at_step), to = last_unit(at_step);
                for (int block = 0; block < slots / 4; ++block) {
                    uint32_t scale_of[kTiles][4], zero_of[kTiles][2] = {};  // (zero points: bytes, those of units 0 and 1, of 2 and 3 in one register)
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        spread(next_scales.scale[t], scale_of[t], at_step, block, t);
                        if constexpr (kZeros) {
                            uint32_t pairs[kDiag];
#pragma unroll
                            for (int d = 0; d < kDiag; ++d) pairs[d] = (next_scales.zero[t][d / 2] >> (16 * (d % 2)) & 0xffu) | (next_scales.zero[t][d / 2] >> (16 * (d % 2)) & 0xff00u) << 8;
                            uint32_t of_unit[4];
                            spread(pairs, of_unit, at_step, block, t);
                            zero_of[t][0] = of_unit[0] | of_unit[1] << 8;
                            zero_of[t][1] = of_unit[2] | of_unit[3] << 8;
                        }
                    }
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        uint32_t scale_pair[kTiles], zero_pair[kTiles];
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) {
                            scale_pair[t] = scale_of[t][a];
                            zero_pair[t] = zero_of[t][a / 2];
                        }
                        const int u = from + block * 4 + a;
                        if (u < to) consume(ring[a % kAhead], u, scale_pair, zero_pair, a % 2);
                        if ((a + kAhead) % 4 == 0) load_scales(next_scales, load_step, load_slot / 4);
                        load_next(ring[a % kAhead]);
                    }
                }
                leave(i);
            }
            finish(first_step + done, number);
            if (done + p.batch < steps) lds_barrier();  // (the results' place is free)
        }
    }
}

// y[t] = sum of its routes' rows, in the order of the slots.  A launch and two trips to memory: 4 to 5 us.
__global__ __launch_bounds__(256) void sum_routes_kernel(const float* rows, const Ids ids, int tokens, int topk, int hidden, bool half, uint16_t* y)
{
    const int per_row = hidden / 4, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= tokens * per_row) return;
    const int token = i / per_row, at = (i - token * per_row) * 4;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int first = 0; first < topk; first += 8) {  // (ids and rows of eight slots are asked for together; rows nobody wrote are not added)
        int expert[8];
        f32x4 row[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int route = token * topk + min(first + i, topk - 1);
            expert[i] = ids[route];
            row[i] = *reinterpret_cast<const f32x4*>(rows + static_cast<size_t>(route) * hidden + at);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i < topk && expert[i] >= 0) sum += row[i];
    }
    uint16_t* const to = y + static_cast<size_t>(token) * hidden + at;
#pragma unroll
    for (int d = 0; d < 4; ++d) to[d] = narrow(sum[d], half);
}

// ---- launches ----------------------------------------------------------------------------------------------------------------------
constexpr int kMaxLds = 160 << 10, kStaticLds = 64;

// Lets a kernel have all of a CU's LDS; once for each device.
template <auto kKernel>
int allow_lds()
{
    constexpr int kMaxDevices = 64;
    static std::atomic<bool> configured[kMaxDevices];
    int device = 0;
    DPEP_HIP(hipGetDevice(&device));
    const bool tracked = device >= 0 && device < kMaxDevices;
    if (!tracked || !configured[device].load(std::memory_order_acquire)) {
        DPEP_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds - kStaticLds));
        if (tracked) configured[device].store(true, std::memory_order_release);
    }
    return DPEP_OK;
}

template <Kind kKind>
int launch_product(Product p, int type, int matrices_most, int rows_expected, int rows_most, hipStream_t stream)
{
    p.units = (p.k + kUnit - 1) / kUnit;
    p.groups = p.k / p.group;
    const int diag = p.group >= 128 ? 1 : 128 / p.group;
    p.group_inverse = diag == 1 ? ((1 << 20) + p.group / 128 - 1) / (p.group / 128) : 0;
    const int tiles = kKind == kMatvec ? 1 : 2, counted = kKind == kGateUp ? p.n / 2 : (p.n + tiles - 1) / tiles;
    p.tile_groups = (counted + 15) / 16;
    p.ragged = p.k % kUnit != 0 || p.group > 128;
    p.split = 1;
    while (p.split < kWaves && p.split * 4 < p.units) p.split *= 2, ++p.log_split;  // (four units to a wave and step)
    const int at_once = kWaves / p.split;
    p.steps = (p.tile_groups + at_once - 1) / at_once;
    const int tokens = 16 / diag, experts = kKind == kMatvec ? 0 : p.ids.local;
    int by_blocks = rows_expected <= tokens ? 1 : 4;
    auto plan = [&](int rows, int batch) { return LdsPlan(p.units, diag, by_blocks, tiles, rows, batch, experts, p.routes, kKind == kGateUp).bytes + kStaticLds; };
    auto rows_in = [&](int limit) {
        int rows = std::min(rows_most, tokens * by_blocks);
        while (rows > (kKind == kDown ? 2 : 1) && plan(rows, 1) > limit) --rows;
        return rows;
    };
    // Four blocks of rows where LDS holds them, with one workgroup to a CU; else one block: with two workgroups, which share the LDS, if the rows that are
    // expected fit half of it, with one if they do not.  (64 rows through 8192 x 8192 and 4096 x 7168 take 61 and 42 us, in four blocks that are never
    // full 112 and 50, with two workgroups 84 and 51; 16 through 4096 x 7168 14.4, with two workgroups 18; 6 through 8192 x 8192 14.5 and 21.)
    if (by_blocks == 4 && rows_in(kMaxLds) <= tokens) by_blocks = 1;
    const bool two = by_blocks == 1 && rows_in(kMaxLds / 2) >= std::min(rows_expected, tokens);
    const int limit = two ? kMaxLds / 2 : kMaxLds;
    int rows = rows_in(limit);
    if (kKind == kDown) rows &= ~1;
    if constexpr (kKind == kMatvec) {
        // A pass waits for its rows, so there are as many passes, even ones of four rows and more, as CUs without work can take (33 rows through
        // 1407 x 2880: 11.5 us, 14.1 in passes of 16, 16 and 1 (10.1 since scales stay in registers); 16 through 2048 x 2048: 7.2 and 10.0; 64 through 512 x 2048: 9.0 and 14.4).
        const int passes = std::max((p.rows + rows - 1) / rows, std::min(256 / p.steps, (p.rows + 3) / 4));
        rows = (p.rows + passes - 1) / passes;
    }
    p.row_cap = rows;
    p.batch = 1;
    while (p.batch < 8 && plan(rows, p.batch + 1) <= limit) ++p.batch;
    const int bytes = plan(rows, p.batch) - kStaticLds;
    const int matrices = kKind == kMatvec ? (p.rows + rows - 1) / rows : matrices_most;
    const long long all_steps = static_cast<long long>(matrices) * p.steps;
    DPEP_REQUIRE(all_steps <= INT32_MAX, "w4: N=%d is too much for %d rows of K=%d", p.n, p.rows, p.k);
    const int grid = static_cast<int>(std::min<long long>(all_steps, two ? 512 : 256));
    int status = DPEP_OK;
    auto go = [&](auto half, auto zeros, auto d, auto b, auto streamed) {
        constexpr auto kernel = product_kernel<kKind, half(), zeros(), d(), b(), streamed()>;
        if (bytes > 32 << 10) status = allow_lds<kernel>();
        if (status != DPEP_OK) return;
        kernel<<<grid, kThreads, bytes, stream>>>(p);
        status = launch_status("w4 product");
    };
    auto by_block = [&](auto half, auto zeros, auto d) {
        // Rows of whole lines are read once and go past the caches; of other rows every other line is read by two waves (through 8 of 256 experts
        // 48 us, plain loads 53; through 4 of 32 with rows of 1440 and 704 bytes 53 and 44).  (A branch around the loads costs a tenth.)
        if (by_blocks == 4) go(half, zeros, d, std::integral_constant<int, 4>{}, std::false_type{});
        else if (p.k % kUnit == 0) go(half, zeros, d, std::integral_constant<int, 1>{}, std::true_type{});
        else go(half, zeros, d, std::integral_constant<int, 1>{}, std::false_type{});
    };
    auto by_group = [&](auto half, auto zeros) {
        if (diag == 1) by_block(half, zeros, std::integral_constant<int, 1>{});
        else if (diag == 2) by_block(half, zeros, std::integral_constant<int, 2>{});
        else by_block(half, zeros, std::integral_constant<int, 4>{});
    };
    auto by_zeros = [&](auto half) {
        if (p.zeros != nullptr) by_group(half, std::true_type{});
        else by_group(half, std::false_type{});
    };
    if (type == DPEP_TYPE_F16) by_zeros(std::true_type{});
    else by_zeros(std::false_type{});
    return status;
}

int check_w4(const dpep_w4* w, int type, const char* what)
{
    DPEP_REQUIRE(w != nullptr, "%s: weights is NULL", what);
    DPEP_REQUIRE(type == DPEP_TYPE_BF16 || type == DPEP_TYPE_F16, "%s: type=%d is neither BF16 nor FP16", what, type);
    DPEP_REQUIRE(w->n >= 1 && w->n <= DPEP_W4_MAX_N && w->k >= 32 && w->k <= kMaxK, "%s: N=%d K=%d: N is at most 2^30, K %d", what, w->n, w->k, kMaxK);
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
    DPEP_REQUIRE(num_rows >= 0 && num_rows <= DPEP_W4_MAX_ROWS, "w4_matvec: num_rows=%d is not in [0, %d]", num_rows, DPEP_W4_MAX_ROWS);
    if (num_rows == 0) return DPEP_OK;
    DPEP_REQUIRE(x != nullptr && y != nullptr && aligned16(x), "w4_matvec: a NULL or misaligned buffer");
    // Workgroups store their columns while others still read rows and weights.
    const size_t of_rows = static_cast<size_t>(num_rows) * 2, groups = static_cast<size_t>(w->n) * (w->k / w->group), y_bytes = of_rows * w->n;
    DPEP_REQUIRE(!overlap(y, y_bytes, x, of_rows * w->k) && !overlap(y, y_bytes, w->packed, static_cast<size_t>(w->n) * (w->k / 2)) &&
                     !overlap(y, y_bytes, w->scales, groups * 2) && !overlap(y, y_bytes, w->zeros, groups),
                 "w4_matvec: y must not overlap x or the weights");
    Product p = {};
    p.packed = w->packed;
    p.scales = static_cast<const uint16_t*>(w->scales);
    p.zeros = w->zeros;
    p.n = w->n;
    p.k = w->k;
    p.group = w->group;
    p.all_scales = static_cast<size_t>(p.n) * (p.k / p.group);
    p.x = static_cast<const uint16_t*>(x);
    p.rows = num_rows;
    p.out = y;
    return launch_product<kMatvec>(p, type, 1, num_rows, num_rows, static_cast<hipStream_t>(stream));
}

size_t dpep_w4_experts_scratch_bytes(int num_tokens, int num_topk, int hidden, int intermediate)
{
    if (num_tokens < 0 || num_topk < 1 || hidden < 1 || intermediate < 1) return 0;
    return static_cast<size_t>(num_tokens) * num_topk * (static_cast<size_t>(intermediate) + hidden) * 4;
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
    // (the sum of the routes reads ids while it stores y; rows and weights have been read by then)
    DPEP_REQUIRE(!overlap(y, static_cast<size_t>(num_tokens) * down->n * 2, topk_idx, static_cast<size_t>(num_tokens) * num_topk * index_bytes),
                 "w4_experts: y must not overlap topk_idx");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int routes = num_tokens * num_topk, slots = std::min(routes, num_local);
    // rows of an expert: about routes / experts, at most all of them (a token may name an expert twice)
    const int expected = 2 * routes / num_local + 1;
    Product p = {};
    p.packed = gate_up->packed;
    p.scales = static_cast<const uint16_t*>(gate_up->scales);
    p.zeros = gate_up->zeros;
    p.n = gate_up->n;
    p.k = gate_up->k;
    p.group = gate_up->group;
    p.all_scales = static_cast<size_t>(num_local) * p.n * (p.k / p.group);
    p.x = static_cast<const uint16_t*>(x);
    p.ids = {topk_idx, index_bytes == 8, expert_begin, num_local};
    p.routes = routes;
    p.topk = num_topk;
    p.route_weights = topk_weights;
    p.out = scratch;
    if (int rc = launch_product<kGateUp>(p, type, slots, expected, routes, s); rc != DPEP_OK) return rc;
    float* const rows = static_cast<float*>(scratch) + static_cast<size_t>(routes) * down->k;
    p.packed = down->packed;
    p.scales = static_cast<const uint16_t*>(down->scales);
    p.zeros = down->zeros;
    p.n = down->n;
    p.k = down->k;
    p.group = down->group;
    p.all_scales = static_cast<size_t>(num_local) * p.n * (p.k / p.group);
    p.x = static_cast<const uint16_t*>(scratch);
    p.out = rows;
    if (int rc = launch_product<kDown>(p, type, slots, 2 * expected, 2 * routes, s); rc != DPEP_OK) return rc;
    const int pieces = num_tokens * (down->n / 4);
    sum_routes_kernel<<<(pieces + 255) / 256, 256, 0, s>>>(rows, p.ids, num_tokens, num_topk, down->n, type == DPEP_TYPE_F16, static_cast<uint16_t*>(y));
    return launch_status("w4_experts");
}

}  // extern "C"
