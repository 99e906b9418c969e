// The matrix product behind the linear cross entropy: out[q][p] = sum over k of P[p,k] Q[q,k], 16-bit operands,
// fp32 sums, on the matrix cores.
//
// A workgroup makes a tile of BP x BQ outputs, WP x WQ wavefronts of it.  Steps of 64 along k go from global
// memory straight into LDS (no registers between), STAGES of them in flight.  An operand lies in memory with its rows
// along k ("along": [row][k]) or across ("across": [k][row]); the second is turned by the LDS's transposing read,
// so no operand is ever copied to turn it.  P is the matrix instruction's first operand: a lane then holds four
// consecutive p of one q, and outputs are stored along p.
//
// An fp32 operand comes as planes of bfloat16 (each the rounded rest of those before it); the sum then runs over
// pairs of planes as well.  16-bit operands have one plane and one pair.
#pragma once

#include "gm_ops.hpp"

namespace gm {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
#define GM_LDS __attribute__((address_space(3)))

template <typename T>
__device__ inline f32x4 multiply_add(s16x8 p, s16x8 q, f32x4 acc);
template <>
__device__ inline f32x4 multiply_add<_Float16>(s16x8 p, s16x8 q, f32x4 acc)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), acc, 0, 0, 0);
}
template <>
__device__ inline f32x4 multiply_add<__bf16>(s16x8 p, s16x8 q, f32x4 acc)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, p), __builtin_bit_cast(b16x8, q), acc, 0, 0, 0);
}

constexpr int kStepK = 64;

struct Operand {
    const short *base;
    int64_t stride;           // elements from row to row of what lies in memory
    int64_t plane;            // elements from plane to plane
    int rows;                 // rows of the product (p or q); memory holds that many, rounded up to 8 when across
};

// Which planes are multiplied: pair i is (P plane, Q plane) = two bits each of codes >> 4 i.
struct PlanePairs {
    int count;
    uint32_t codes;
};

// One operand's share of a step: ROWS rows by kStepK, brought in by all wavefronts together, sixteen bytes a lane.
// In LDS, along: 128 bytes a row in eight pieces of 16; piece c of row r lies at c ^ (r & 7), so that the sixteen
// rows a fragment read touches lie on different banks.  Across: 2 ROWS bytes a k in pieces of 32 (sixteen rows); piece g of
// k lies at g ^ f(k), f taking eight values over the k that one read touches, for the same reason.
template <int ROWS, bool ACROSS, int WAVES>
struct Tile {
    static constexpr int kBytes = ROWS * kStepK * 2;
    static constexpr int kLoads = kBytes / 1024 / WAVES;         // per wavefront
    static_assert(kLoads * 1024 * WAVES == kBytes, "whole loads");
    static constexpr int kPieces = ROWS / 16;                    // across: pieces of 32 bytes a k

    __device__ static inline int across_swizzle(int k) { return ((k & 3) | ((k >> 1) & 4)) & (kPieces - 1); }

    // This lane's source addresses for one step, k0 the step's first k, `limit` the k that exist (across).
    __device__ static inline void load(const Operand &op, const short *plane, int row0, int k0, int limit, uint32_t lds, int wave, int lane)
    {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int at = (i * WAVES + wave) * 1024 + lane * 16;      // byte of the tile this lane fills
            const short *src;
            if (!ACROSS) {
                const int row = at / 128, piece = ((at / 16) & 7) ^ (row & 7);
                const int r = row0 + row < op.rows ? row0 + row : op.rows - 1;
                src = plane + (int64_t)r * op.stride + k0 + piece * 8;
            } else {
                const int k = at / (ROWS * 2), half = (at / 16) & 1, group = ((at / 32) & (kPieces - 1)) ^ across_swizzle(k);
                const int last = (op.rows - 1) & ~7;      // (rows are there in eights)
                int r = row0 + group * 16 + half * 8;
                r = r < last ? r : last;
                const int kk = k0 + k < limit ? k0 + k : limit - 1;
                src = plane + (int64_t)kk * op.stride + r;
            }
            const uint32_t to = lds + (i * WAVES + wave) * 1024;
            // (m0 takes the wavefront's LDS address; one wait state lies between its write and its use)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(src) : "memory");
        }
    }

    // The fragment of rows row .. row + 15, k half * 32 .. + 31: lane l has row l % 16, k 8 (l / 16) .. + 7 of them.
    __device__ static inline s16x8 fragment(uint32_t lds, int row, int half, int lane)
    {
        if (!ACROSS) {
            const int r = row + (lane & 15), c = half * 4 + (lane >> 4);
            return *reinterpret_cast<const GM_LDS s16x8 *>(lds + r * 128 + ((c ^ (r & 7)) << 4));
        }
        s16x8 out;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int k = half * 32 + (lane >> 4) * 8 + j * 4 + ((lane & 15) >> 2);
            const int group = (row >> 4) ^ across_swizzle(k);
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                reinterpret_cast<GM_LDS s16x4 *>(lds + k * (ROWS * 2) + (group << 5) + (lane & 3) * 8));
#pragma unroll
            for (int e = 0; e < 4; e++) out[j * 4 + e] = v[e];
        }
        return out;
    }
};

// Workgroups go round the eight XCDs, each with an L2 of its own: consecutive tiles are given to one XCD.  Within them
// runs of `group` tiles along q share a tile of P.  false: no tile for this workgroup.
__device__ inline bool tile_of(uint32_t block, uint32_t tiles_p, uint32_t tiles_q, uint32_t group, uint32_t &tp, uint32_t &tq)
{
    const uint32_t total = tiles_p * tiles_q, per = (total + 7) / 8;
    const uint32_t local = block / 8, t = (block & 7) * per + local;
    if (local >= per || t >= total) return false;
    const uint32_t in_group = group * tiles_p, g = t / in_group, rest = t - g * in_group;
    const uint32_t height = tiles_q - g * group < group ? tiles_q - g * group : group;
    tp = rest / height;
    tq = g * group + rest - tp * height;
    return true;
}

template <int BP_, int BQ_, int WP_, int WQ_, int STAGES_>
struct Shape {
    static constexpr int BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, STAGES = STAGES_;
    static constexpr int WAVES = WP * WQ, THREADS = WAVES * 64;
    static constexpr int MP = BP / WP / 16, MQ = BQ / WQ / 16;        // matrix instructions a wavefront, either way
    static constexpr int LDS = (BP + BQ) * kStepK * 2 * STAGES;
};

// The sum over steps [first, last) of the pairs' k; acc[i][j]: rows 16 i of P, 16 j of Q of this wavefront.
// steps: steps of one pair; limit_p / limit_q: the k that exist where an operand lies across.
template <typename T, typename S, bool PACROSS, bool QACROSS>
__device__ inline void multiply_tiles(const Operand &p, const Operand &q, const PlanePairs &pairs, int p0, int q0, int steps, int limit_p,
                                      int limit_q, int first, int last, uint32_t lds, f32x4 (&acc)[S::MP][S::MQ])
{
    typedef Tile<S::BP, PACROSS, S::WAVES> TP;
    typedef Tile<S::BQ, QACROSS, S::WAVES> TQ;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave / S::WQ * (S::BP / S::WP), wq = wave % S::WQ * (S::BQ / S::WQ);
#pragma unroll
    for (int i = 0; i < S::MP; i++)
#pragma unroll
        for (int j = 0; j < S::MQ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const auto load = [&](int step) {      // beyond the last step the last one again, into a stage that nobody reads
        const int s = step < last ? step : last - 1;
        const int pair = s / steps, k0 = (s - pair * steps) * kStepK;
        const uint32_t code = pairs.codes >> (4 * pair);
        const uint32_t at = lds + (uint32_t)((step - first) % S::STAGES) * (TP::kBytes + TQ::kBytes);
        TP::load(p, p.base + (int64_t)(code & 3) * p.plane, p0, k0, limit_p, at, wave, lane);
        TQ::load(q, q.base + (int64_t)(code >> 2 & 3) * q.plane, q0, k0, limit_q, at + TP::kBytes, wave, lane);
    };
    for (int s = 0; s < S::STAGES - 1; s++) load(first + s);
    for (int step = first; step < last; step++) {
        // this step's loads have arrived (those of the later stages may be on their way), and every wavefront is done
        // with the stage that is filled next
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S::STAGES - 2) * (TP::kLoads + TQ::kLoads)) : "memory");
        __builtin_amdgcn_s_barrier();
        load(step + S::STAGES - 1);
        const uint32_t at = lds + (uint32_t)((step - first) % S::STAGES) * (TP::kBytes + TQ::kBytes);
#pragma unroll
        for (int half = 0; half < 2; half++) {
            s16x8 fp[S::MP], fq[S::MQ];
#pragma unroll
            for (int j = 0; j < S::MQ; j++) fq[j] = TQ::fragment(at + TP::kBytes, wq + j * 16, half, lane);
#pragma unroll
            for (int i = 0; i < S::MP; i++) fp[i] = TP::fragment(at, wp + i * 16, half, lane);
#pragma unroll
            for (int i = 0; i < S::MP; i++)
#pragma unroll
                for (int j = 0; j < S::MQ; j++) acc[i][j] = multiply_add<T>(fp[i], fq[j], acc[i][j]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}

}  // namespace gm
