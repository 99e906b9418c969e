// The matrix product behind the linear cross entropy: out[q][p] = sum over k of P[p,k] Q[q,k], 16-bit operands,
// fp32 sums, on the matrix cores.
//
// A workgroup makes a tile of BP x BQ outputs, WP x WQ wavefronts of it.  Steps of 64 along k go from global
// memory straight into LDS (no registers between), STAGES of them in flight.  An operand lies in memory with its rows
// along k ("along": [row][k]) or across ("across": [k][row]); the second is turned by the LDS's transposing read,
// so no operand is ever copied to turn it.  P is the matrix instruction's first operand: a lane then holds four
// consecutive p of one q, and outputs are stored along p.
//
// An operand of more bits comes as planes (each the rounded rest of those before it); the sum then runs over pairs of planes
// as well.  16-bit operands have one plane and one pair.
#pragma once

#include "gm_ops.hpp"

#include <type_traits>

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

    // Byte offsets of this lane's loads from the tile's first k of row 0, rows behind the last one replaced by it.
    __device__ static inline void offsets(const Operand &op, int row0, int wave, int lane, uint32_t (&out)[kLoads])
    {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int at = (i * WAVES + wave) * 1024 + lane * 16;      // byte of the tile this lane fills
            if (!ACROSS) {
                const int row = at / 128, piece = ((at / 16) & 7) ^ (row & 7);
                const int r = row0 + row < op.rows ? row : op.rows - 1 - row0;
                out[i] = (uint32_t)r * (uint32_t)op.stride * 2u + piece * 16;
            } else {
                const int k = at / (ROWS * 2), half = (at / 16) & 1, group = ((at / 32) & (kPieces - 1)) ^ across_swizzle(k);
                const int last = (op.rows - 1) & ~7;                   // (rows are there in eights)
                const int r = row0 + group * 16 + half * 8;
                out[i] = (uint32_t)k * (uint32_t)op.stride * 2u + (uint32_t)((r < last ? r : last) - row0) * 2u;
            }
        }
    }

    // The last step of a sum that is no whole number of steps: `there` of its k exist, the others become the last one again
    // (across; along, rows are whole steps long).
    __device__ static inline void clamp(int there, uint32_t stride_bytes, int wave, int lane, uint32_t (&out)[kLoads])
    {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int k = ((i * WAVES + wave) * 1024 + lane * 16) / (ROWS * 2);
            if (k >= there) out[i] -= (uint32_t)(k - there + 1) * stride_bytes;
        }
    }

    // The wavefront's i-th load of a step.  `base`: the tile's first k of row 0.
    __device__ static inline void load(const char *base, uint32_t offset, uint32_t lds, int wave, int i)
    {
        // (m0 takes the wavefront's LDS address, as an operand that the compiler writes there; one wait state lies between its
        // write and its use)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(lds + (i * WAVES + wave) * 1024), "v"(offset), "s"(base) : "memory");
    }

    // Where this lane reads the fragments of the wavefront's rows row .. row + 16 N - 1: lane l has row l % 16 and k 8 (l / 16)
    // .. + 7 of a half.  Along, the fragments of a half lie a constant apart; across, every sixteen rows have a place.
    template <int N>
    struct Places {
        uint32_t at[ACROSS ? N : 2];
    };
    template <int N>
    __device__ static inline Places<N> places(uint32_t lds, int row, int lane)
    {
        Places<N> out;
        if (!ACROSS) {
            const int r = row + (lane & 15);
#pragma unroll
            for (int half = 0; half < 2; half++) out.at[half] = lds + r * 128 + (((half * 4 + (lane >> 4)) ^ (r & 7)) << 4);
        } else {
            const int k = (lane >> 4) * 8 + ((lane & 15) >> 2);
#pragma unroll
            for (int i = 0; i < N; i++) out.at[ACROSS ? i : 0] = lds + k * (ROWS * 2) + (((row / 16 + i) ^ across_swizzle(k)) << 5) + (lane & 3) * 8;
        }
        return out;
    }
    template <int N>
    __device__ static inline void move(Places<N> &places, uint32_t bytes)      // to the next stage
    {
#pragma unroll
        for (int i = 0; i < (ACROSS ? N : 2); i++) places.at[i] += bytes;
    }
    template <int N>
    __device__ static inline s16x8 fragment(const Places<N> &places, int i, int half)
    {
        if (!ACROSS) return *reinterpret_cast<const GM_LDS s16x8 *>(places.at[half] + (uint32_t)(i * 2048));
        s16x8 out;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                reinterpret_cast<GM_LDS s16x4 *>(places.at[ACROSS ? i : 0] + (uint32_t)(half * (32 * ROWS * 2) + j * (4 * ROWS * 2))));
#pragma unroll
            for (int e = 0; e < 4; e++) out[j * 4 + e] = v[e];
        }
        return out;
    }
};

// Workgroups go round the eight XCDs, each with an L2 of its own: consecutive pieces of work are given to one XCD.  They are
// the tiles of one part of the sum after those of another, and within a part runs of `group` tiles along q share a
// tile of P.  false: nothing for this workgroup.
__device__ inline bool tile_of(uint32_t block, uint32_t tiles_p, uint32_t tiles_q, uint32_t parts, uint32_t group, uint32_t &tp, uint32_t &tq,
                               uint32_t &part)
{
    const uint32_t tiles = tiles_p * tiles_q, total = tiles * parts, per = (total + 7) / 8;
    const uint32_t local = block / 8, w = (block & 7) * per + local;
    if (local >= per || w >= total) return false;
    part = w / tiles;
    const uint32_t t = w - part * tiles;
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
    static constexpr int LDS = (BP + BQ) * kStepK * 2 * STAGES;       // bytes of all stages
    static constexpr int TURN = WQ * BP * 16 * 4;                     // bytes that turn_rows takes
    static_assert(TURN <= LDS, "turning rows fits the stages' memory");
};

// The sum over steps [first, last) of the pairs' k for one tile; acc[i][j]: rows 16 i of P, 16 j of Q of this wavefront.
// steps: steps of one pair; limit_p / limit_q: the k that exist where an operand lies across.
//
// A step's matrix instructions come in two halves of 32 k, row by row of P's fragments.  A fragment of P is replaced by
// the next half's as soon as its row is through, so reads from LDS run half a step ahead all the time.  Shortly after the
// first half every wavefront has read all of its stage: one barrier there frees the stage for the loads of the step
// STAGES later, and makes the next step's data, which have arrived by then, visible.
//
template <typename T, typename S, bool PACROSS, bool QACROSS>
struct Multiplier {
    typedef Tile<S::BP, PACROSS, S::WAVES> TP;
    typedef Tile<S::BQ, QACROSS, S::WAVES> TQ;
    static constexpr int kLoads = TP::kLoads + TQ::kLoads;
    static constexpr int kMeet = S::MP >= 4 ? 1 : 0;      // the row of the second half that the barrier follows
    // Q's fragments are all needed by the next half's first row: they are read behind the first rows
    static constexpr int kEarly = S::MP >= 2 * S::MQ ? 1 : S::MP >= S::MQ ? 2 : S::MQ;

    const Operand p, q;
    const PlanePairs pairs;
    const int steps, limit_p, limit_q, first, last, edge;      // edge: the k of a pair's last step; steps may run past the last pair's
                                                               // end and go on at the first one's beginning
    const uint32_t lds, lds_q;                                 // P's stages, then Q's
    const int lane, wave;
    int p0, q0;
    uint32_t off_p[TP::kLoads], off_q[TQ::kLoads];
    int load_step, load_pair, load_k;                          // the next step to load
    const char *from_p, *from_q;

    __device__ inline Multiplier(const Operand &p_, const Operand &q_, const PlanePairs &pairs_, int steps_, int limit_p_, int limit_q_, int first_,
                                 int last_, uint32_t lds_)
        : p(p_), q(q_), pairs(pairs_), steps(steps_), limit_p(limit_p_), limit_q(limit_q_), first(first_), last(last_), edge((steps_ - 1) * kStepK),
          lds(lds_), lds_q(lds_ + S::STAGES * TP::kBytes), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6))
    {
    }

    __device__ inline void seek()
    {
        const uint32_t code = pairs.codes >> (4 * load_pair);
        const short *bp = p.base + (int64_t)(code & 3) * p.plane, *bq = q.base + (int64_t)(code >> 2 & 3) * q.plane;
        from_p = reinterpret_cast<const char *>(PACROSS ? bp + (int64_t)load_k * p.stride + p0 : bp + (int64_t)p0 * p.stride + load_k);
        from_q = reinterpret_cast<const char *>(QACROSS ? bq + (int64_t)load_k * q.stride + q0 : bq + (int64_t)q0 * q.stride + load_k);
    }
    __device__ inline void at_edge()
    {
        if (PACROSS && limit_p < edge + kStepK) TP::clamp(limit_p - edge, (uint32_t)p.stride * 2u, wave, lane, off_p);
        if (QACROSS && limit_q < edge + kStepK) TQ::clamp(limit_q - edge, (uint32_t)q.stride * 2u, wave, lane, off_q);
    }
    __device__ inline void load_one(int stage, int i)      // i: which of this wavefront's loads
    {
        if (i < TP::kLoads) TP::load(from_p, off_p[i < TP::kLoads ? i : 0], lds + stage * TP::kBytes, wave, i);
        else TQ::load(from_q, off_q[i >= TP::kLoads ? i - TP::kLoads : 0], lds_q + stage * TQ::kBytes, wave, i - TP::kLoads);
    }
    __device__ inline void loaded()
    {
        load_step++;
        load_k += kStepK;
        from_p += PACROSS ? (int64_t)p.stride * (2 * kStepK) : 2 * kStepK;
        from_q += QACROSS ? (int64_t)q.stride * (2 * kStepK) : 2 * kStepK;
        if (load_k >= edge) {
            if (load_k > edge) {      // the next pair from its beginning
                load_k = 0;
                load_pair = load_pair + 1 < pairs.count ? load_pair + 1 : 0;
                seek();
                if (PACROSS && limit_p < edge + kStepK) TP::offsets(p, p0, wave, lane, off_p);
                if (QACROSS && limit_q < edge + kStepK) TQ::offsets(q, q0, wave, lane, off_q);
            }
            if (load_k == edge) at_edge();
        }
    }

    // Every wavefront of the workgroup must be done with the tiles in LDS.
    __device__ inline void start(int p0_, int q0_)
    {
        p0 = p0_, q0 = q0_;
        TP::offsets(p, p0, wave, lane, off_p);
        TQ::offsets(q, q0, wave, lane, off_q);
        load_step = first, load_pair = first / steps, load_k = (first - load_pair * steps) * kStepK;
        seek();
        if (load_k == edge) at_edge();
#pragma unroll
        for (int s = 0; s < S::STAGES; s++)
            if (load_step < last) {
#pragma unroll
                for (int i = 0; i < kLoads; i++) load_one(s, i);
                loaded();
            }
    }

    // Where turn_rows may work for this wavefront, after run().
    __device__ inline uint32_t turn_place() const { return lds + wave * (S::BP / S::WP * 16 * 4); }

    __device__ inline void run(f32x4 (&acc)[S::MP][S::MQ])
    {
        const int wp = wave / S::WQ * (S::BP / S::WP), wq = wave % S::WQ * (S::BQ / S::WQ);
        auto at_p = TP::template places<S::MP>(lds, wp, lane);
        auto at_q = TQ::template places<S::MQ>(lds_q, wq, lane);
#pragma unroll
        for (int i = 0; i < S::MP; i++)
#pragma unroll
            for (int j = 0; j < S::MQ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (first + S::STAGES <= last) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S::STAGES - 1) * kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();

        s16x8 fp[S::MP], fq[2][S::MQ];
        // The order is pinned (sched_barrier): left to itself the compiler gathers the reads in front of their first use, and the
        // matrix cores wait for them.
        const auto row = [&](int half, int i) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < S::MQ; j++) acc[i][j] = multiply_add<T>(fp[i], fq[half][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        };
        int stage = 0;
        // `more`: a step is left to load, and all stages are under way
        const auto whole_step = [&](auto more) {
#pragma unroll
            for (int i = 0; i < S::MP; i++) {      // the first half; the second one's fragments are read
                row(0, i);
#pragma unroll
                for (int j = i * kEarly; j < (i + 1) * kEarly && j < S::MQ; j++) fq[1][j] = TQ::fragment(at_q, j, 1);
                fp[i] = TP::fragment(at_p, i, 1);
            }
            const bool wraps = stage == S::STAGES - 1;
            TP::move(at_p, wraps ? -(S::STAGES - 1) * TP::kBytes : TP::kBytes);
            TQ::move(at_q, wraps ? -(S::STAGES - 1) * TQ::kBytes : TQ::kBytes);
#pragma unroll
            for (int i = 0; i < S::MP; i++) {      // the second half; the next step's first half is read
                row(1, i);
                if (i < kMeet) continue;
                if (i == kMeet) {
                    if constexpr (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S::STAGES - 2) * kLoads) : "memory");
                    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                }
                constexpr int kRows = S::MP - kMeet;
                const int at = i - kMeet;
#pragma unroll
                for (int j = at * kEarly; j < (at + 1) * kEarly && j < S::MQ; j++) fq[0][j] = TQ::fragment(at_q, j, 0);
#pragma unroll
                for (int r = i == kMeet ? 0 : i; r <= i; r++) fp[r] = TP::fragment(at_p, r, 0);
                if constexpr (more) {
#pragma unroll
                    for (int l = at * kLoads / kRows; l < (at + 1) * kLoads / kRows; l++) load_one(stage, l);
                }
            }
            if constexpr (more) loaded();
            stage = wraps ? 0 : stage + 1;
        };
#pragma unroll
        for (int j = 0; j < S::MQ; j++) fq[0][j] = TQ::fragment(at_q, j, 0);
#pragma unroll
        for (int i = 0; i < S::MP; i++) fp[i] = TP::fragment(at_p, i, 0);
        int step = first;
        for (; step + S::STAGES < last; step++) whole_step(std::true_type());
        for (; step < last; step++) whole_step(std::false_type());
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();      // everyone is done with the tiles
    }
};

// Sixteen rows of Q's outputs go through the wavefront's own share of LDS on their way out: a lane holds four p of one q,
// and what it would store is 8 bytes of each of sixteen rows; turned, a wavefront stores whole rows of its p, 16 bytes a
// lane.  `use(row, p, v)` gets eight consecutive p (from the wavefront's first) of row 0 .. 15.  Pieces of 16 bytes of
// row r lie at their number XOR r, so that neither side meets on a bank.  mine: memory of this wavefront's own.
template <typename S>
constexpr int kTurnRows = 64 / (S::BP / S::WP / 8);

template <typename S, typename F>
__device__ inline void turn_rows(uint32_t mine, const f32x4 (&v)[S::MP], F &&use)
{
    constexpr int kSpan = S::BP / S::WP, kPitch = kSpan * 4, kLanes = kSpan / 8, kRows = kTurnRows<S>, kMask = kSpan / 4 - 1 < 15 ? kSpan / 4 - 1 : 15;
    const int lane = threadIdx.x & 63, to = lane & 15;
#pragma unroll
    for (int i = 0; i < S::MP; i++)
        *reinterpret_cast<GM_LDS f32x4 *>(mine + to * kPitch + (((i * 4 + (lane >> 4)) ^ (to & kMask)) << 4)) = v[i];
#pragma unroll
    for (int pass = 0; pass < 16 / kRows; pass++) {
        const int row = pass * kRows + lane / kLanes, piece = lane % kLanes * 2;
        const f32x4 a = *reinterpret_cast<const GM_LDS f32x4 *>(mine + row * kPitch + ((piece ^ (row & kMask)) << 4));
        const f32x4 b = *reinterpret_cast<const GM_LDS f32x4 *>(mine + row * kPitch + (((piece + 1) ^ (row & kMask)) << 4));
        float out[8];
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = a[e], out[4 + e] = b[e];
        use(row, piece * 4, out);
    }
}

}  // namespace gm
