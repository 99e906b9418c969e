// Softmax cross entropy of a linear output layer over a large vocabulary, with its gradients, without the logits.
//
//   s = x W^T          loss_i = lse(s_i) - s_i[t_i]          dS = (exp(s - lse) - onehot(t)) c
//   dX = dS W          dW (+)= dS^T x                        c = gradient scale * loss scale (/ counted tokens)
//
// Tokens whose target is the ignored one (or no word of the vocabulary) take no part: the others are packed first,
// so they cost nothing and whatever stands in them reaches no sum.  Then, for as many tokens at a time as the
// workspace holds:
//   logits_kernel   a tile of logits stays in registers: of each token's share of a tile its maximum m and the sum of
//                   exp(s - m) are kept, the target's logit in fp32, and (gradients wanted) exp(s - m) itself
//   rows_kernel     one token a workgroup: lse from its tiles' maxima and sums, the loss, and exp(s - m) turned into dS
//                   (the target's entry as expm1 of its fp32 logit: p - 1 of a certain token keeps its digits)
//   product_kernel  dX and dW
// 2 N V D operations each: the product of the logits is made once and not again for the gradients; what it costs is
// the pass of rows_kernel over the workspace.
// What bounds them: the matrix cores (at the clock the card's power leaves them) the three products, memory rows_kernel and the packing,
// and for up to 128 tokens the stream of the weights.  4096 x 131072 x 4096 fp16, one token in ten ignored: logits 3.3,
// rows 0.39 (1.9 GB, 4.9 TB/s), dX 3.06, dW 3.08 ms, 1.2 to 1.3 PFLOP/s; one bf16 token, 131072 x 4096: logits 182 us, 5.9 TB/s.
// 513 x 10007 x 1000 fp32: packing 27, logits 60, rows 13, dX 45 + 9 (joining its parts), dW 51 us.
#include "gm_matrix.hpp"

#include "../../include/gometal_hip.h"

#include <cmath>

namespace gm {

// What the kernels of one call find out on the device.
struct LossHead {
    int count;                 // tokens that take part
    float coefficient;         // c above
    int x_exponent, w_exponent;      // the largest of the rows' exponents (operands with a scale for each row)
};

typedef Shape<256, 256, 2, 4, 2> WideShape;       // products of many tiles: 128 KiB of LDS, one workgroup a CU
typedef Shape<128, 128, 2, 2, 2> SquareShape;     // fewer tiles than a wide shape needs to fill the chip
typedef Shape<256, 128, 4, 2, 3> TallShape;       // up to 128 tokens: the weights' stream bounds it, three steps of it in flight
typedef Shape<128, 32, 4, 1, 4> FlatShape;        // up to 32 tokens: the weights' stream is all there is
enum : int { kWide, kSquare, kTall, kFlat };
constexpr int kShapeP[4] = {256, 128, 256, 128}, kShapeQ[4] = {256, 128, 128, 32}, kShapeSpan[4] = {128, 64, 64, 32};

// exp(s - m) in 16 bits is 32768 times itself in fp16, dS of fp16 operands 16384 times itself: both keep clear of the
// subnormals (down to 2^-29 and 2^-28), and each of an entry's two roundings is at most 2^-11 of it (the second one 2^-8 with bf16).
// 4096 x 131072 x 4096 fp16: gradients are 2.4e-4 off the formula, of which the rounding of the outputs alone makes 2.1e-4; exponentials
// kept in 32 bits would spare the first of the two at twice the bytes that the logits write and rows_kernel reads.
constexpr float kExpScale = 32768.0f, kExpShift = 15.0f;
template <typename T>
constexpr float kSlopeScale = 1.0f;
template <>
constexpr float kSlopeScale<_Float16> = 16384.0f;

// Operands with a scale for each row.  fp32 tensors are multiplied as two parts of fp16 (h, and what is left of the value after
// h) with the products h h, h l and l h: 22 bits and a bit, about what fp32 sums keep of the result.  fp16's short range is made up
// for by the rows' own powers of two: a row whose largest element lies below 2^e is taken times 2^(15 - e), so that a part's
// least step, 2^-24, is 2^-39 of the row's largest.  The logits' epilogue undoes both rows' powers.  Where a row's index is
// what the sum runs over (W's in dX, X's in dW) its power goes into dS, relative to the largest row's; there are two sets of dS
// then.  (Three parts of bfloat16 with six products need no scales, and took twice the matrix work: 513 x 10007 x 1000 in 293 us.)
// bfloat16 activations are one such part, for a weight gradient in fp32: with dS in two parts that is two products, with
// bfloat16 parts of dS it were three.
constexpr int kRowBits = 15, kSlopeBits = 14;

__device__ inline int chunk_rows(const LossHead *head, int first, int most)
{
    const int left = head->count - first;
    return left < 0 ? 0 : left < most ? left : most;
}

// ------------------------------------------------------------------------------------------ tokens that count ----
constexpr int kScanBlock = 1024;

__device__ inline void write_head(LossHead *head, int count, int mean, float gradient_scale, const AmpScaleView &amp)
{
    float scale = gradient_scale;
    if (amp.scale[0]) scale = scale * *amp.scale[*amp.stamp[1] > *amp.stamp[0] ? 1 : 0];
    head->count = count;
    head->coefficient = mean ? scale / (float)(count > 0 ? count : 1) : scale;
}

// Packs the tokens that take part: row_of[r] is the r-th one, place_of[i] where token i went (-1: nowhere).
__global__ void __launch_bounds__(kScanBlock)
scan_targets_kernel(const int *targets, int n, int vocab, int ignore, int mean, float gradient_scale, AmpScaleView amp, LossHead *head,
                    int *row_of, int *place_of, int *row_target)
{
    __shared__ int of_wave[kScanBlock / 64 + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int done = 0;
    for (int base = 0; base < n; base += kScanBlock) {
        const int i = base + (int)threadIdx.x;
        const int t = i < n ? targets[i] : ignore;
        const bool counts = i < n && t != ignore && (unsigned)t < (unsigned)vocab;
        const unsigned long long votes = __ballot(counts);
        if (lane == 0) of_wave[wave] = __popcll(votes);
        __syncthreads();
        if (threadIdx.x == 0) {
            int sum = 0;
            for (int w = 0; w < kScanBlock / 64; w++) {
                const int c = of_wave[w];
                of_wave[w] = sum;
                sum += c;
            }
            of_wave[kScanBlock / 64] = sum;
        }
        __syncthreads();
        const int place = done + of_wave[wave] + __popcll(votes & ((1ull << lane) - 1ull));
        if (i < n) place_of[i] = counts ? place : -1;
        if (counts) {
            row_of[place] = i;
            row_target[place] = t;
        }
        done += of_wave[kScanBlock / 64];
        __syncthreads();
    }
    if (threadIdx.x == 0) write_head(head, done, mean, gradient_scale, amp);
}

// Eight elements as the planes of an operand: rounded to nearest, then what is left of them after that, and so on.
template <typename T>
__device__ inline void split_store(float (&v)[8], T *to, int64_t plane, int planes)
{
    for (int k = 0; k < planes; k++) {
        store8(to + k * plane, true, 8, v);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = v[e] - (float)from_float<T>(v[e]);
    }
}

// Eight elements of a matrix's row of `dim`, zeros behind it.
template <typename I>
__device__ inline void load_padded(const I *row, int c, int dim, bool aligned, float (&v)[8])
{
    const int count = dim - c < 8 ? (dim - c < 0 ? 0 : dim - c) : 8;
    load8(row + c, aligned && count == 8, count, v);
}

// The same for a row of an operand.  Of two parts an element that is not finite takes the second, with 0 for the first: of the other
// operand it then meets the first part alone.  In both, or in the first, it would meet the other's second part as well, whose sign or
// zero makes NaN of an infinite logit (a word that a bias of -inf bans).
__device__ inline void split_operand(float (&v)[8], _Float16 *to, int64_t plane, int planes)
{
    if (planes != 2) return split_store<_Float16>(v, to, plane, planes);
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        rest[e] = v[e];
        v[e] = fabsf(v[e]) < INFINITY ? v[e] : 0.0f;
    }
    store8(to, true, 8, v);
#pragma unroll
    for (int e = 0; e < 8; e++) rest[e] = rest[e] - (float)from_float<_Float16>(v[e]);
    store8(to + plane, true, 8, rest);
}

// The power of two of a row: its largest finite element lies below 2^e (for a row without one but zero less than any other's, so that
// it takes no part in the largest).  One wavefront; the same in all lanes.
template <typename I>
__device__ inline int row_exponent(const I *row, int dim, bool aligned)
{
    const int lane = threadIdx.x & 63;
    uint32_t top = 0;
    for (int c = lane * 8; c < dim; c += 64 * 8) {
        float v[8];
        load_padded(row, c, dim, aligned, v);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t bits = __float_as_uint(v[e]) & 0x7FFFFFFFu;
            top = bits < 0x7F800000u && bits > top ? bits : top;
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const uint32_t other = (uint32_t)__shfl_xor((int)top, o);
        top = top > other ? top : other;
    }
    if (top == 0) return -200;
    int e = 0;
    (void)frexpf(__uint_as_float(top), &e);
    return e;
}

__device__ inline void scale8(float (&v)[8], int e)
{
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = ldexpf(v[k], e);
}

constexpr int kPackBlock = 256;

// Up to this many tokens every workgroup of pack_tokens_kernel counts the ones before its own by itself: a launch less, 2 to 3 us.
constexpr int kCountedTokens = 2048;

struct PackArgs {
    int64_t x_stride, packed_stride, plane, dx_stride;      // plane: of the scaled rows
    bool aligned;
    int n, dim, width;
    int first;              // the launch's first workgroup
    bool plain;             // the rows as they are
    // COUNT: what scan_targets_kernel does otherwise
    const int *targets;
    int vocab, ignore, mean;
    float gradient_scale;
    AmpScaleView amp;
    int *row_of, *row_target;
    // operand rows with a scale each
    int scaled_planes;
    _Float16 *scaled;
    short *exponents;       // by packed token
};

// Workgroup i < n: token i's activations to their place, or zeros to its outputs.  The rows behind the last counted
// token, up to a whole step of k, become zeros.
template <typename I, typename T, bool COUNT>
__global__ void __launch_bounds__(kPackBlock)
pack_tokens_kernel(PackArgs a, const I *x, LossHead *head, const int *place_of, T *packed, float *losses, I *dx)
{
    __shared__ int of_wave[kPackBlock / 64];
    const int i = a.first + (int)blockIdx.x;
    int place, count;
    if (COUNT) {
        // the counted tokens before i (all of them, for the workgroups behind the last token)
        int mine = 0;
        for (int j = threadIdx.x; j < (i < a.n ? i : a.n); j += kPackBlock) {
            const int t = a.targets[j];
            mine += t != a.ignore && (unsigned)t < (unsigned)a.vocab;
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) mine += __shfl_xor(mine, o);
        if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = mine;
        __syncthreads();
        place = 0;
#pragma unroll
        for (int w = 0; w < kPackBlock / 64; w++) place += of_wave[w];
        count = place;
        if (i == a.n && threadIdx.x == 0) write_head(head, count, a.mean, a.gradient_scale, a.amp);
        if (i < a.n) {
            const int t = a.targets[i];
            if (t == a.ignore || (unsigned)t >= (unsigned)a.vocab) {
                place = -1;
            } else if (threadIdx.x == 0) {
                a.row_of[place] = i;
                a.row_target[place] = t;
            }
        }
    } else {
        place = i < a.n ? place_of[i] : -1;
        count = head->count;
    }
    if (i >= a.n) {
        const int r = count + (i - a.n), end = (count + kStepK - 1) / kStepK * kStepK;
        float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (r < end)
            for (int c = threadIdx.x * 8; c < a.width; c += kPackBlock * 8) {
                if (a.plain) store8(packed + r * a.packed_stride + c, true, 8, zero);
                split_store<_Float16>(zero, a.scaled + r * a.packed_stride + c, a.plane, a.scaled_planes);
            }
        return;
    }
    if (place >= 0) {
        const I *row = x + i * a.x_stride;
        int exponent = 0;
        if (a.scaled_planes) {
            exponent = row_exponent(row, a.dim, a.aligned);
            if (threadIdx.x == 0) a.exponents[place] = (short)exponent;
        }
        for (int c = threadIdx.x * 8; c < a.width; c += kPackBlock * 8) {
            float v[8];
            load_padded(row, c, a.dim, a.aligned, v);
            if (a.plain) store8(packed + place * a.packed_stride + c, true, 8, v);
            if (a.scaled_planes) {
                scale8(v, kRowBits - exponent);
                split_operand(v, a.scaled + place * a.packed_stride + c, a.plane, a.scaled_planes);
            }
        }
        return;
    }
    if (threadIdx.x == 0) losses[i] = 0.0f;
    if (dx)
        for (int c = threadIdx.x; c < a.dim; c += kPackBlock) dx[i * a.dx_stride + c] = (I)0.0f;
}

// The weights as operand rows of `width` elements (a multiple of 64), eight a lane.
template <typename I, typename T>
__global__ void __launch_bounds__(kPackBlock)
pack_weights_kernel(const I *w, int64_t w_stride, bool aligned, int rows, int dim, int width, T *packed)
{
    const int per_row = width / 8;
    const int64_t first = (int64_t)blockIdx.x * kPackBlock;
    const int first_row = (int)(first / per_row), at = (int)(first - (int64_t)first_row * per_row) + (int)threadIdx.x;
    const int row = first_row + at / per_row, c = at % per_row * 8;
    if (row >= rows) return;
    float v[8];
    load_padded(w + row * w_stride, c, dim, aligned, v);
    store8(packed + (int64_t)row * width + c, true, 8, v);
}

// fp32 weights as two parts of fp16, a scale for each row; a wavefront a row.
__global__ void __launch_bounds__(kPackBlock)
pack_scaled_weights_kernel(const float *w, int64_t w_stride, bool aligned, int rows, int dim, int width, _Float16 *packed, int64_t plane,
                           short *exponents)
{
    const int row = blockIdx.x * (kPackBlock / 64) + (threadIdx.x >> 6);
    if (row >= rows) return;
    const float *from = w + row * w_stride;
    const int exponent = row_exponent(from, dim, aligned);
    if ((threadIdx.x & 63) == 0) exponents[row] = (short)exponent;
    for (int c = (threadIdx.x & 63) * 8; c < width; c += 64 * 8) {
        float v[8];
        load_padded(from, c, dim, aligned, v);
        scale8(v, kRowBits - exponent);
        split_operand(v, packed + (int64_t)row * width + c, plane, 2);
    }
}

// The largest of the rows' exponents; one workgroup.  (Every row's workgroup raising one word took 90 us for 10007 rows.)
__global__ void __launch_bounds__(1024)
largest_exponents_kernel(LossHead *head, const short *x, const short *w, int words)
{
    __shared__ int of_wave[2][16];
    int top[2] = {-100000, -100000};
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const short *from = k ? w : x;
        const int n = k ? words : head->count;
        for (int i = threadIdx.x * 8; i < n; i += 1024 * 8) {      // (the arrays are there in eights)
            const s16x8 v = *reinterpret_cast<const s16x8 *>(from + i);
#pragma unroll
            for (int e = 0; e < 8; e++) top[k] = i + e < n && v[e] > top[k] ? v[e] : top[k];
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const int other = __shfl_xor(top[k], o);
            top[k] = top[k] > other ? top[k] : other;
        }
        if ((threadIdx.x & 63) == 0) of_wave[k][threadIdx.x >> 6] = top[k];
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        int most = -100000;
        for (int wave = 0; wave < 16; wave++) most = most > of_wave[threadIdx.x][wave] ? most : of_wave[threadIdx.x][wave];
        (threadIdx.x ? head->w_exponent : head->x_exponent) = most;
    }
}

// --------------------------------------------------------------------------------------------------- logits ----
enum : int { kKeepNothing, kKeepHalf, kKeepFloat };

struct LogitsArgs {
    Operand w, x;               // x: the chunk's rows
    PlanePairs pairs;
    int steps, first, most, vocab, padded;      // padded: vocab up to a whole step of k
    const LossHead *head;
    const int *row_target;      // by packed token
    float *target_logit;
    float2 *stats;              // [row of the chunk][group]: maximum, sum of exp(s - maximum)
    int groups, keep;
    void *kept;                 // [row of the chunk][stride]
    int64_t stride;
    const short *x_exponents, *w_exponents;      // nullptr: rows have no scales of their own.  Of w's, whole tiles are there
};

template <typename T, typename S>
__global__ void __launch_bounds__(S::THREADS)
logits_kernel(LogitsArgs a)
{
    __shared__ __attribute__((aligned(1024))) char tiles[S::LDS];
    const int rows = chunk_rows(a.head, a.first, a.most);
    uint32_t tp, tq, part;
    if (!tile_of(blockIdx.x, (a.vocab + S::BP - 1) / S::BP, (rows + S::BQ - 1) / S::BQ, 1, 8, tp, tq, part)) return;
    a.x.rows = rows;
    const int p0 = (int)tp * S::BP, q0 = (int)tq * S::BQ;
    f32x4 acc[S::MP][S::MQ];
    const uint32_t lds = (uint32_t)(uintptr_t)(GM_LDS char *)tiles;
    // One tile of tokens: nobody shares the weights' rows, and every workgroup begins at a k of its own.  At one k the rows of all
    // tiles, a power of two apart, lie on one channel: 128 x 65536 x 4096, 537 MB of weights, 165 -> 135 us.  (Up to 32 tokens,
    // where tiles are half as high and four steps are in flight, it gains nothing: 203 -> 207 us for one token.)
    const int first = rows <= S::BQ && S::BQ > 32 ? (int)(tp * 5 % (uint32_t)a.steps) : 0;
    Multiplier<T, S, false, false> product(a.w, a.x, a.pairs, a.steps, 0, 0, first, first + a.steps * a.pairs.count, lds);
    product.start(p0, q0);
    product.run(acc);      // (from here on the stages' memory turns rows)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wp = p0 + wave / S::WQ * (S::BP / S::WP) + (lane >> 4) * 4, wq = q0 + wave % S::WQ * (S::BQ / S::WQ) + (lane & 15);
    const int group = (p0 + wave / S::WQ * (S::BP / S::WP)) / (S::BP / S::WP);
    const bool ragged = p0 + S::BP > a.vocab;
    if (a.w_exponents) {
#pragma unroll
        for (int j = 0; j < S::MQ; j++) {
            const int by = (wq + j * 16 < rows ? a.x_exponents[a.first + wq + j * 16] : 0) - 2 * kRowBits;
#pragma unroll
            for (int i = 0; i < S::MP; i++) {
                const s16x4 e = *reinterpret_cast<const s16x4 *>(a.w_exponents + wp + i * 16);
#pragma unroll
                for (int r = 0; r < 4; r++) acc[i][j][r] = ldexpf(acc[i][j][r], e[r] + by);
            }
        }
    }
    // what this lane stores of the exponentials: always the same eight words
    const int wave_q = wq - (lane & 15), turn_col = wp - (lane >> 4) * 4 + lane % (64 / kTurnRows<S>) * 8;
    char *kept = static_cast<char *>(a.kept) + (wave_q * a.stride + turn_col) * (a.keep == kKeepFloat ? 4 : 2);
#pragma unroll
    for (int j = 0; j < S::MQ; j++) {
        const int q = wq + j * 16;
        const bool there = q < rows;
        // the target's logit, if it is one of this lane's: words wp + 16 i + (0 .. 3)
        const int at = (there ? a.row_target[a.first + q] : -1) - wp;
        if (at >= 0 && at < S::MP * 16 && (at & 15) < 4) {
            float logit = 0.0f;
#pragma unroll
            for (int i = 0; i < S::MP; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) logit = at == i * 16 + r ? acc[i][j][r] : logit;
            a.target_logit[a.first + q] = logit;
        }
        if (ragged) {
#pragma unroll
            for (int i = 0; i < S::MP; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[i][j][r] = wp + i * 16 + r < a.vocab ? acc[i][j][r] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < S::MP; i++) top = fmaxf(fmaxf(fmaxf(top, acc[i][j][0]), acc[i][j][1]), fmaxf(acc[i][j][2], acc[i][j][3]));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float ref = top == -INFINITY ? 0.0f : top;      // (a share that lies behind the vocabulary: all zeros)
        float sum = 0.0f;
        f32x4 v[S::MP];
        if (a.keep == kKeepFloat) {
#pragma unroll
            for (int i = 0; i < S::MP; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) sum += v[i][r] = expf(acc[i][j][r] - ref);
        } else {
            // 2^15 exp(s - ref) by the hardware's power of two; the sum's factor is taken out again exactly
#pragma unroll
            for (int i = 0; i < S::MP; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) sum += v[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r] - ref, 1.44269504f, kExpShift));
            sum *= 1.0f / kExpScale;
        }
        if (a.keep != kKeepNothing)
            turn_rows<S>(product.turn_place(), v, [&](int row, int, const float (&e)[8]) {
                const int to = j * 16 + row;
                if (turn_col >= a.padded || wave_q + to >= rows) return;
                if (a.keep == kKeepFloat) store8(reinterpret_cast<float *>(kept) + to * a.stride, true, 8, e);
                else store8(reinterpret_cast<_Float16 *>(kept) + to * a.stride, true, 8, e);
            });
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (there && lane < 16) a.stats[(int64_t)q * a.groups + group] = float2{top, sum};
    }
}

// ----------------------------------------------------------------------------------------------------- rows ----
constexpr int kRowBlock = 512;

struct RowsArgs {
    int first, most, vocab, padded, groups, span;       // span: words of a group
    const LossHead *head;
    const int *row_of, *row_target;
    const float *target_logit;
    const float2 *stats;
    float *losses;
    int keep, planes;
    void *kept, *slopes;       // kKeepHalf: the same memory
    int64_t stride, plane;
    // operands with scales: of w's rows for these slopes (nullptr: none), and a second set, for dW, with x's rows' (0 planes: none)
    const short *w_exponents, *x_exponents;
    int dw_planes;
    _Float16 *dw_slopes;
};

__device__ inline float block_reduce(float x, bool maximum, float *scratch)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const float y = __shfl_xor(x, o);
        x = maximum ? fmaxf(x, y) : x + y;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    x = scratch[0];
#pragma unroll
    for (int w = 1; w < kRowBlock / 64; w++) x = maximum ? fmaxf(x, scratch[w]) : x + scratch[w];
    return x;
}

template <typename T>
__global__ void __launch_bounds__(kRowBlock)
rows_kernel(RowsArgs a)
{
    __shared__ float scratch[kRowBlock / 64];
    const int rows = chunk_rows(a.head, a.first, a.most), r = blockIdx.x;
    T *slopes = static_cast<T *>(a.slopes) + r * a.stride;
    const float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (r >= rows) {
        if (a.keep != kKeepNothing && r < (rows + kStepK - 1) / kStepK * kStepK)      // a whole step of k for dW
            for (int c = threadIdx.x * 8; c < a.padded; c += kRowBlock * 8) {
                for (int k = 0; k < a.planes; k++) store8(slopes + k * a.plane + c, true, 8, zero);
                for (int k = 0; k < a.dw_planes; k++) store8(a.dw_slopes + r * a.stride + k * a.plane + c, true, 8, zero);
            }
        return;
    }
    const float2 *stats = a.stats + (int64_t)r * a.groups;
    float top = -INFINITY;
    for (int g = threadIdx.x; g < a.groups; g += kRowBlock) top = fmaxf(top, stats[g].x);
    top = block_reduce(top, true, scratch);
    float sum = 0.0f;
    for (int g = threadIdx.x; g < a.groups; g += kRowBlock) sum += stats[g].y * expf(stats[g].x - top);
    sum = block_reduce(sum, false, scratch);
    const float lse = top + logf(sum), target_logit = a.target_logit[a.first + r];
    if (threadIdx.x == 0) a.losses[a.row_of[a.first + r]] = lse - target_logit;
    if (a.keep == kKeepNothing) return;
    const int target = a.row_target[a.first + r];
    const float at_target = expm1f(target_logit - lse);
    const int w_shift = a.w_exponents ? kSlopeBits - a.head->w_exponent : 0;
    const int x_shift = a.dw_planes ? a.x_exponents[a.first + r] - a.head->x_exponent + kSlopeBits : 0;
    for (int c = threadIdx.x * 8; c < a.padded; c += kRowBlock * 8) {
        float v[8];
        float f = c < a.vocab ? expf(stats[c / a.span].x - lse) : 0.0f;
        if (a.keep == kKeepHalf) {
            load8(static_cast<const _Float16 *>(a.kept) + r * a.stride + c, true, 8, v);
            f = f * (1.0f / kExpScale);
        } else {
            load8(static_cast<const float *>(a.kept) + r * a.stride + c, true, 8, v);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = c + e < a.vocab ? (c + e == target ? at_target : v[e] * f) : 0.0f;
        if (a.dw_planes) {
            float scaled[8];
#pragma unroll
            for (int e = 0; e < 8; e++) scaled[e] = ldexpf(v[e], x_shift);
            split_store<_Float16>(scaled, a.dw_slopes + r * a.stride + c, a.plane, a.dw_planes);
        }
        if (a.w_exponents) {
            const s16x8 e8 = *reinterpret_cast<const s16x8 *>(a.w_exponents + c);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = ldexpf(v[e], e8[e] + w_shift);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = v[e] * kSlopeScale<T>;
        }
        split_store<T>(v, slopes + c, a.plane, a.planes);
    }
}

// The sum (or mean) of the losses and the number of tokens that count; one workgroup, sums in 64 bits in a fixed order.  (A launch
// of its own: with the last of rows_kernel's workgroups doing it, the counting of all of them cost more, 3 us at 64 tokens
// and 60 us at 4096.)
__global__ void __launch_bounds__(1024)
total_kernel(const float *losses, int n, int mean, const LossHead *head, float *loss)
{
    __shared__ double part[1024];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) sum += (double)losses[i];
    part[threadIdx.x] = sum;
    for (int o = 512; o; o >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    }
    if (threadIdx.x == 0) {
        const int count = head->count;
        loss[0] = (float)(mean ? part[0] / (double)(count > 0 ? count : 1) : part[0]);
        loss[1] = (float)count;
    }
}

// ------------------------------------------------------------------------------------------------- products ----
struct ProductArgs {
    Operand p, q;
    PlanePairs pairs;
    int first, most;                 // the chunk's tokens
    int steps;                       // steps of 64 k of one pair; 0: as many as the chunk has tokens (dW)
    int limit_p;                     // across: the k that exist
    int splits;                      // parts of the sum; more than one: `partial` takes them
    float *partial;                  // [split][partial_rows][p rows]
    int partial_rows;                // at least as many as q has
    const LossHead *head;
    const int *row_of;               // dX: where a packed row belongs
    float unscale;                   // undoes kSlopeScale
    const int *exponent;             // of the largest row, where rows have scales (nullptr: they have none)
    void *out;
    int64_t out_stride;
    int out_type;
    int accumulate;                  // add what `out` holds
    const float *add;                // and this, of out's shape without gaps (nullptr: nothing)
    bool out_aligned;                // rows of out begin at multiples of 16 bytes
    bool skip_empty;                 // a chunk without tokens leaves `out` alone
};

template <typename O>
__device__ inline void finish_as(const ProductArgs &a, O *out, int64_t row, int p, float (&v)[8])
{
    const int count = a.p.rows - p < 8 ? a.p.rows - p : 8;
    const bool whole = a.out_aligned && count == 8;
    O *at = out + row * a.out_stride + p;
    if (a.accumulate) {
        float old[8];
        load8(at, whole, count, old);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = old[e] + v[e];
    }
    store8(at, whole, count, v);
}

// What the sums are multiplied by: a factor, then a power of two, apart: small rows' power by itself may lie below the least
// fp32 number where the output does not.
struct Factor {
    float by;
    int power;
    __device__ inline float operator()(float v) const { return ldexpf(v * by, power); }
};

__device__ inline Factor output_factor(const ProductArgs &a)
{
    return Factor{a.head->coefficient * a.unscale, a.exponent ? *a.exponent - kRowBits - kSlopeBits : 0};
}

// Eight outputs of one row: times c, added to what is there, rounded once.
__device__ inline void finish(const ProductArgs &a, const Factor &by, int q, int p, float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = by(v[e]);
    if (a.add) {
        const int count = a.p.rows - p < 8 ? a.p.rows - p : 8;
        float more[8];
        load8(a.add + (int64_t)q * a.p.rows + p, count == 8 && a.p.rows % 4 == 0, count, more);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = more[e] + v[e];
    }
    const int64_t row = a.row_of ? a.row_of[a.first + q] : q;
    if (a.out_type == kFloat32) finish_as(a, static_cast<float *>(a.out), row, p, v);
    else if (a.out_type == kFloat16) finish_as(a, static_cast<_Float16 *>(a.out), row, p, v);
    else finish_as(a, static_cast<__bf16 *>(a.out), row, p, v);
}

// The wavefront's outputs, all of which exist, to rows that begin at multiples of 16 bytes: nothing is left of finish() but
// the product and the rounding.  (With its cases the stores of a tile took more time than 128 tokens' matrix work.)
template <typename S, typename O>
__device__ inline void store_whole(O *out, int64_t stride, const Factor &by, uint32_t turn, const f32x4 (&acc)[S::MP][S::MQ])
{
    const int lane = threadIdx.x & 63;
    constexpr int kLanes = 64 / kTurnRows<S>;
    O *at = out + (lane / kLanes) * stride + lane % kLanes * 8;
#pragma unroll
    for (int j = 0; j < S::MQ; j++) {
        f32x4 v[S::MP];
#pragma unroll
        for (int i = 0; i < S::MP; i++) v[i] = acc[i][j];
        turn_rows<S>(turn, v, [&](int, int, float (&o)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = by(o[e]);
            store8(at, true, 8, o);
            at += kTurnRows<S> * stride;
        });
    }
}

// The tile at (p0, q0) out of the workgroup's accumulators.
template <typename S>
__device__ inline void store_tile(const ProductArgs &a, const Factor &by, int p0, int q0, uint32_t split, uint32_t turn, const f32x4 (&acc)[S::MP][S::MQ])
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave_p = p0 + wave / S::WQ * (S::BP / S::WP), wave_q = q0 + wave % S::WQ * (S::BQ / S::WQ);
    if (wave_p + S::BP / S::WP <= a.p.rows && wave_q + S::BQ / S::WQ <= a.q.rows) {
        if (a.splits > 1 && a.p.rows % 4 == 0) {
            store_whole<S>(a.partial + ((int64_t)split * a.partial_rows + wave_q) * a.p.rows + wave_p, a.p.rows, Factor{1.0f, 0}, turn, acc);
            return;
        }
        if (a.splits == 1 && a.out_aligned && !a.accumulate && !a.add && !a.row_of) {
            const int64_t at = wave_q * a.out_stride + wave_p;
            if (a.out_type == kFloat32) store_whole<S>(static_cast<float *>(a.out) + at, a.out_stride, by, turn, acc);
            else if (a.out_type == kFloat16) store_whole<S>(static_cast<_Float16 *>(a.out) + at, a.out_stride, by, turn, acc);
            else store_whole<S>(static_cast<__bf16 *>(a.out) + at, a.out_stride, by, turn, acc);
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < S::MQ; j++) {
        if (wave_q + j * 16 >= a.q.rows) break;
        f32x4 v[S::MP];
#pragma unroll
        for (int i = 0; i < S::MP; i++) v[i] = acc[i][j];
        turn_rows<S>(turn, v, [&](int row, int p, float (&out)[8]) {
            const int q = wave_q + j * 16 + row;
            p += wave_p;
            if (q >= a.q.rows || p >= a.p.rows) return;
            if (a.splits > 1) {
                const int count = a.p.rows - p < 8 ? a.p.rows - p : 8;
                store8(a.partial + ((int64_t)split * a.partial_rows + q) * a.p.rows + p, count == 8 && a.p.rows % 4 == 0, count, out);
            } else {
                finish(a, by, q, p, out);
            }
        });
    }
}

// DW: Q is dS across and the sum runs over the chunk's tokens; otherwise dX, Q is dS along.  P lies across in both.
template <typename T, typename S, bool DW>
__global__ void __launch_bounds__(S::THREADS)
product_kernel(ProductArgs a)
{
    __shared__ __attribute__((aligned(1024))) char tiles[S::LDS];
    const int rows = chunk_rows(a.head, a.first, a.most);
    if (rows == 0 && (!DW || a.skip_empty)) return;
    if (DW) a.steps = (rows + kStepK - 1) / kStepK;
    else a.q.rows = rows;
    const uint32_t tiles_p = (a.p.rows + S::BP - 1) / S::BP, tiles_q = (a.q.rows + S::BQ - 1) / S::BQ;
    uint32_t tp, tq, split;
    if (!tile_of(blockIdx.x, tiles_p, tiles_q, a.splits, 8, tp, tq, split)) return;
    const int limit = DW ? a.steps * kStepK : a.limit_p;
    const int total = a.steps * a.pairs.count;
    const int begin = (int)((int64_t)total * split / a.splits), end = (int)((int64_t)total * (split + 1) / a.splits);
    const int p0 = (int)tp * S::BP, q0 = (int)tq * S::BQ;
    Multiplier<T, S, true, DW> product(a.p, a.q, a.pairs, a.steps, limit, limit, begin, end, (uint32_t)(uintptr_t)(GM_LDS char *)tiles);
    f32x4 acc[S::MP][S::MQ];
    if (begin < end) {
        product.start(p0, q0);
        product.run(acc);
    } else {      // a chunk without tokens that dW has to be written for all the same
#pragma unroll
        for (int i = 0; i < S::MP; i++)
#pragma unroll
            for (int j = 0; j < S::MQ; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    store_tile<S>(a, output_factor(a), p0, q0, split, product.turn_place(), acc);
}

// The parts of a split sum, added up in order; eight outputs a lane.
__global__ void __launch_bounds__(256)
join_splits_kernel(ProductArgs a)
{
    const int tokens = chunk_rows(a.head, a.first, a.most), rows = a.row_of ? tokens : a.q.rows;
    if (tokens == 0 && a.skip_empty) return;
    const int per_row = (a.p.rows + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int q = (int)(i / per_row), p = (int)(i - (int64_t)q * per_row) * 8;
    if (q >= rows) return;
    const int count = a.p.rows - p < 8 ? a.p.rows - p : 8;
    const bool whole = count == 8 && a.p.rows % 4 == 0;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kAhead = 4;
    for (int s = 0; s < a.splits; s += kAhead) {
        float v[kAhead][8];
#pragma unroll
        for (int k = 0; k < kAhead; k++) load8(a.partial + ((int64_t)(s + k < a.splits ? s + k : s) * a.partial_rows + q) * a.p.rows + p, whole, count, v[k]);
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (s + k < a.splits) {
#pragma unroll
                for (int e = 0; e < 8; e++) sum[e] += v[k][e];
            }
    }
    finish(a, output_factor(a), q, p, sum);
}

// ------------------------------------------------------------------------------------------------ host side ----
// Everything that follows from the sizes: what lies where in the workspace, and which shape each product takes.
struct LossPlan {
    int n, vocab, dim, width, padded, chunk, chunks;
    int x_stride, slope_stride;            // of the packed tokens and of dS
    bool plain;                            // x (and W, if it is packed) as it is
    int scaled_planes;                     // and with a scale for each row
    int slope_planes, dw_slope_planes, keep;      // of dS; of its second set, for dW
    bool gradients, pack_weights, sum_weights;      // sum_weights: dW of several chunks in 16 bits needs fp32 sums
    int logits_shape, groups, dx_shape, dx_splits, dw_shape, dw_splits;
    size_t head, row_of, place_of, row_target, target_logit, x, scaled_x, x_exponents, w, w_exponents, stats, kept, slopes, dw_slopes, partial, sums, bytes;
};

// Rows that the kernels lay out themselves are 128 bytes longer than their contents: a step reads 128 bytes of 256 rows, and
// rows a large power of two apart would all lie on the same channel of the L2.
constexpr int kSkew = 64;

constexpr int kLeastChunk = 256;
constexpr size_t kKeptBytes = (size_t)4 << 30;      // of exp(s - m) and dS together, unless one chunk needs more

// A launch can address fewer than 2^32 lanes.  Packing goes in launches of at most so many workgroups; a token of rows_kernel takes 512
// lanes and a tile of 128 x 128 outputs 256, so a chunk has at most kMostChunk tokens, and none of the products more than
// kMostOutputs outputs (2^23 such tiles; ragged edges add less than a tenth).
constexpr int kMostGroups = 1 << 23, kMostChunk = 1 << 22;
constexpr int64_t kMostOutputs = (int64_t)1 << 37;

static int tiles(int shape, int64_t p, int64_t q)      // (below 2^24 for what the plans ask)
{
    return (int)(((p + kShapeP[shape] - 1) / kShapeP[shape]) * ((q + kShapeQ[shape] - 1) / kShapeQ[shape]));
}

// Whether wide tiles finish first.  They come in rounds of 256, one a CU; square ones in rounds of 512, two a CU, that take 0.83
// of a wide round (a quarter of the outputs each, at 0.6 of the rate: their fragments are read from LDS twice as often).
// 300 x 30000 x 1024 fp32, logits: 236 wide tiles 184 us, 705 square ones 210 us; dW of 10007 x 1000: 160 wide tiles instead of
// 632 square ones take 20 us off 100.
static int wide_or_square(int64_t p, int64_t q)
{
    const int wide = (tiles(kWide, p, q) + 255) / 256, square = (tiles(kSquare, p, q) + 511) / 512;
    return wide * 100 <= square * 83 ? kWide : kSquare;
}

static int shape_for(int64_t p, int64_t q)
{
    return q <= kShapeQ[kFlat] ? kFlat : q <= kShapeQ[kTall] ? kTall : wide_or_square(p, q);
}

static LossPlan loss_plan(int n, int vocab, int dim, bool weights_fit, int data_type, int gradient_type, bool gradients, int chunk)
{
    const auto up = [](size_t v, size_t to) { return (v + to - 1) / to * to; };
    LossPlan s{};
    s.n = n, s.vocab = vocab, s.dim = dim, s.gradients = gradients;
    s.width = (int)up((size_t)dim, kStepK), s.padded = (int)up((size_t)vocab, kStepK);
    s.x_stride = s.width + kSkew, s.slope_stride = s.padded + kSkew;
    const bool exact = gradients && gradient_type == kFloat32;      // an fp32 weight gradient
    s.plain = data_type != kFloat32;
    s.scaled_planes = data_type == kFloat32 ? 2 : data_type == kBFloat16 && exact ? 1 : 0;
    s.slope_planes = data_type == kFloat32 || (data_type == kFloat16 && exact) ? 2 : 1;
    s.dw_slope_planes = s.scaled_planes && gradients ? 2 : 0;
    s.keep = !gradients ? kKeepNothing : exact ? kKeepFloat : kKeepHalf;
    s.pack_weights = data_type == kFloat32 || !weights_fit;
    const size_t entry = s.keep == kKeepNothing ? 0 : s.keep == kKeepHalf ? 2 : 4 + 2 * (s.slope_planes + s.dw_slope_planes);
    if (chunk <= 0) {
        size_t most = kMostOutputs / (vocab > dim ? vocab : dim) / kLeastChunk * kLeastChunk;
        if (most > kMostChunk) most = kMostChunk;
        if (entry && most > kKeptBytes / (entry * s.slope_stride)) most = kKeptBytes / (entry * s.slope_stride) / kLeastChunk * kLeastChunk;
        if (most < kLeastChunk) most = kLeastChunk;
        chunk = most < (size_t)n ? (int)most : n;
    }
    s.chunk = chunk < n ? chunk : (n > 0 ? n : 1);
    s.chunks = n > 0 ? (n + s.chunk - 1) / s.chunk : 1;
    s.sum_weights = gradients && s.chunks > 1 && gradient_type != kFloat32;
    s.logits_shape = shape_for(vocab, s.chunk);
    s.groups = (vocab + kShapeP[s.logits_shape] - 1) / kShapeP[s.logits_shape] * (kShapeP[s.logits_shape] / kShapeSpan[s.logits_shape]);
    if (gradients) {
        // few outputs, a long sum: parts of it until every CU has work (two workgroups of the smaller shapes fit a CU), as
        // long as a part is worth a tile's beginning and end; wide tiles where their parts fill the chip
        const auto split = [](int &shape, int &splits, int64_t p, int64_t q, int steps) {
            const auto parts = [&](int of) {
                const int want = (of == kWide || of == kTall ? 256 : 512) / tiles(of, p, q), most = steps / 16;
                return want < 1 || most < 1 ? 1 : want < most ? want : most;
            };
            if (shape == kSquare && tiles(kWide, p, q) * parts(kWide) >= 192) shape = kWide;
            splits = parts(shape);
        };
        s.dx_shape = shape_for(dim, s.chunk);
        split(s.dx_shape, s.dx_splits, dim, s.chunk, s.padded / kStepK * (s.scaled_planes == 2 ? 3 : 1));
        s.dw_shape = wide_or_square(dim, vocab);
        split(s.dw_shape, s.dw_splits, dim, vocab, (s.chunk + kStepK - 1) / kStepK * (s.scaled_planes == 2 ? 3 : s.dw_slope_planes ? 2 : s.slope_planes));
    }
    const size_t rows = up((size_t)n, kStepK), chunk_rows = up((size_t)s.chunk, kStepK);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up(bytes, 256);
        return here;
    };
    s.head = take(sizeof(LossHead));
    s.row_of = take(4 * rows), s.place_of = take(4 * rows), s.row_target = take(4 * rows), s.target_logit = take(4 * rows);
    s.x = take(s.plain ? rows * s.x_stride * 2 : 0);
    s.scaled_x = take(rows * s.x_stride * 2 * s.scaled_planes);
    s.x_exponents = take(s.scaled_planes ? 2 * rows : 0);
    s.w = take(s.pack_weights ? (size_t)vocab * s.width * 2 * (data_type == kFloat32 ? 2 : 1) : 0);
    s.w_exponents = take(data_type == kFloat32 ? 2 * up((size_t)vocab, 256) : 0);      // whole tiles of words
    s.stats = take(sizeof(float2) * (size_t)s.chunk * s.groups);
    s.kept = take(s.keep == kKeepNothing ? 0 : chunk_rows * s.slope_stride * (s.keep == kKeepHalf ? 2 : 4));
    s.slopes = s.keep == kKeepFloat ? take(chunk_rows * s.slope_stride * 2 * s.slope_planes) : s.kept;
    s.dw_slopes = take(chunk_rows * s.slope_stride * 2 * s.dw_slope_planes);
    // (dX is joined before dW's parts are written)
    const size_t dx_parts = gradients && s.dx_splits > 1 ? (size_t)s.dx_splits * s.chunk * dim * 4 : 0;
    const size_t dw_parts = gradients && s.dw_splits > 1 ? (size_t)s.dw_splits * vocab * dim * 4 : 0;
    s.partial = take(dx_parts > dw_parts ? dx_parts : dw_parts);
    s.sums = take(s.sum_weights ? (size_t)vocab * dim * 4 : 0);
    s.bytes = at;
    return s;
}

// The plan with the most tokens at a time that fits the workspace; otherwise the one that needs the fewest bytes.  (That need not be the
// one with the fewest tokens: in 16 bits a weight gradient of several chunks takes fp32 sums of its size.)
static bool fitting_plan(LossPlan &s, size_t bytes, int n, int vocab, int dim, bool weights_fit, int data_type, int gradient_type,
                         bool gradients)
{
    LossPlan next = loss_plan(n, vocab, dim, weights_fit, data_type, gradient_type, gradients, 0);
    s = next;
    while (next.bytes > bytes && next.chunk > kLeastChunk) {
        const int half = (next.chunk / 2 + kLeastChunk - 1) / kLeastChunk * kLeastChunk;
        next = loss_plan(n, vocab, dim, weights_fit, data_type, gradient_type, gradients, half < next.chunk ? half : kLeastChunk);
        if (next.bytes <= bytes || next.bytes < s.bytes) s = next;
    }
    return s.bytes <= bytes;
}

static bool weights_fit(uintptr_t weight, int dim, int stride, int data_type)
{
    return data_type != kFloat32 && weight != 0 && weight % 16 == 0 && dim % kStepK == 0 && stride % 8 == 0 && stride <= 1 << 22;
}

// Codes: P plane + 4 Q plane; the small products first.
static constexpr PlanePairs kOnePair = {1, 0x0};
static constexpr PlanePairs kBothParts = {3, 0x041};      // l h, h l, h h
static constexpr PlanePairs kPartsOfQ = {2, 0x04};        // h l, h h where P has one plane

struct LossCall {
    uintptr_t hidden, weight, targets, losses, loss, dx, dw;
    int hidden_stride, weight_stride, dx_stride, dw_stride, data_type, gradient_type, ignore, mean, accumulate;
    float gradient_scale;
    AmpScaleView amp;
    char *space;
};

template <typename T>
static void launch_logits(int shape, const LogitsArgs &a, int rows, hipStream_t stream)
{
    const int grid = (tiles(shape, a.vocab, rows) + 7) / 8 * 8;
    if (shape == kWide) logits_kernel<T, WideShape><<<grid, WideShape::THREADS, 0, stream>>>(a);
    else if (shape == kSquare) logits_kernel<T, SquareShape><<<grid, SquareShape::THREADS, 0, stream>>>(a);
    else if (shape == kTall) logits_kernel<T, TallShape><<<grid, TallShape::THREADS, 0, stream>>>(a);
    else logits_kernel<T, FlatShape><<<grid, FlatShape::THREADS, 0, stream>>>(a);
}

template <typename T, bool DW>
static void launch_product(int shape, const ProductArgs &a, int p, int q, hipStream_t stream)
{
    const unsigned grid = ((unsigned)tiles(shape, p, q) * a.splits + 7) / 8 * 8;
    if (shape == kWide) product_kernel<T, WideShape, DW><<<grid, WideShape::THREADS, 0, stream>>>(a);
    else if (shape == kSquare) product_kernel<T, SquareShape, DW><<<grid, SquareShape::THREADS, 0, stream>>>(a);
    else if constexpr (!DW) {
        if (shape == kTall) product_kernel<T, TallShape, DW><<<grid, TallShape::THREADS, 0, stream>>>(a);
        else product_kernel<T, FlatShape, DW><<<grid, FlatShape::THREADS, 0, stream>>>(a);
    }
    if (a.splits > 1) join_splits_kernel<<<(unsigned)(((int64_t)q * ((p + 7) / 8) + 255) / 256), 256, 0, stream>>>(a);
}

// I: what the caller's tensors hold; T: what the matrix cores take.
template <typename I, typename T>
static void launch_loss(const LossCall &c, const LossPlan &s, hipStream_t stream)
{
    char *space = c.space;
    LossHead *head = reinterpret_cast<LossHead *>(space + s.head);
    int *row_of = reinterpret_cast<int *>(space + s.row_of), *place_of = reinterpret_cast<int *>(space + s.place_of);
    int *row_target = reinterpret_cast<int *>(space + s.row_target);
    float *target_logit = reinterpret_cast<float *>(space + s.target_logit);
    T *x = reinterpret_cast<T *>(space + s.x);
    float *losses = reinterpret_cast<float *>(c.losses);
    const size_t rows = ((size_t)s.n + kStepK - 1) / kStepK * kStepK, chunk_rows = ((size_t)s.chunk + kStepK - 1) / kStepK * kStepK;
    const int64_t x_plane = (int64_t)rows * s.x_stride, w_plane = (int64_t)s.vocab * s.width, slope_plane = (int64_t)chunk_rows * s.slope_stride;

    _Float16 *scaled_x = reinterpret_cast<_Float16 *>(space + s.scaled_x);
    short *x_exponents = reinterpret_cast<short *>(space + s.x_exponents), *w_exponents = reinterpret_cast<short *>(space + s.w_exponents);
    constexpr bool kFull = std::is_same<I, float>::value;      // fp32: every operand has scales
    const int *targets = reinterpret_cast<const int *>(c.targets);
    PackArgs pack{c.hidden_stride, s.x_stride, x_plane, c.dx_stride, c.hidden % 16 == 0 && c.hidden_stride * sizeof(I) % 16 == 0, s.n, s.dim, s.width, 0,
                        s.plain, targets, s.vocab, c.ignore, c.mean, c.gradient_scale, c.amp, row_of, row_target, s.scaled_planes, scaled_x,
                        x_exponents};
    const I *hidden = reinterpret_cast<const I *>(c.hidden);
    I *dx = reinterpret_cast<I *>(c.dx);
    if (s.n <= kCountedTokens) {
        pack_tokens_kernel<I, T, true><<<s.n + kStepK, kPackBlock, 0, stream>>>(pack, hidden, head, place_of, x, losses, dx);
    } else {
        scan_targets_kernel<<<1, kScanBlock, 0, stream>>>(targets, s.n, s.vocab, c.ignore, c.mean, c.gradient_scale, c.amp, head, row_of,
                                                          place_of, row_target);
        for (; pack.first < s.n + kStepK; pack.first += kMostGroups) {
            const int left = s.n + kStepK - pack.first;
            pack_tokens_kernel<I, T, false><<<left < kMostGroups ? left : kMostGroups, kPackBlock, 0, stream>>>(pack, hidden, head, place_of, x, losses, dx);
        }
    }
    Operand w{reinterpret_cast<const short *>(c.weight), c.weight_stride, 0, s.vocab};
    const bool w_aligned = c.weight % 16 == 0 && c.weight_stride * sizeof(I) % 16 == 0;
    if constexpr (kFull) {
        pack_scaled_weights_kernel<<<(s.vocab + kPackBlock / 64 - 1) / (kPackBlock / 64), kPackBlock, 0, stream>>>(
            reinterpret_cast<const float *>(c.weight), c.weight_stride, w_aligned, s.vocab, s.dim, s.width,
            reinterpret_cast<_Float16 *>(space + s.w), w_plane, w_exponents);
    } else if (s.pack_weights) {
        const int rows_each = (int)((int64_t)kMostGroups * kPackBlock / (s.width / 8));
        for (int first = 0; first < s.vocab; first += rows_each) {
            const int rows = s.vocab - first < rows_each ? s.vocab - first : rows_each;
            const unsigned grid = (unsigned)(((int64_t)rows * (s.width / 8) + kPackBlock - 1) / kPackBlock);
            pack_weights_kernel<I, T><<<grid, kPackBlock, 0, stream>>>(reinterpret_cast<const I *>(c.weight) + (int64_t)first * c.weight_stride,
                                                                       c.weight_stride, w_aligned, rows, s.dim, s.width,
                                                                       reinterpret_cast<T *>(space + s.w) + (int64_t)first * s.width);
        }
    }
    if (s.dw_slope_planes) largest_exponents_kernel<<<1, 1024, 0, stream>>>(head, x_exponents, w_exponents, kFull ? s.vocab : 0);
    if (s.pack_weights) w = Operand{reinterpret_cast<const short *>(space + s.w), s.width, w_plane, s.vocab};
    const PlanePairs pairs = kFull ? kBothParts : kOnePair;
    for (int k = 0; k < s.chunks; k++) {
        const int first = k * s.chunk, most = s.n - first < s.chunk ? s.n - first : s.chunk;
        if (most <= 0 && k > 0) break;
        const Operand plain{reinterpret_cast<const short *>(x + (int64_t)first * s.x_stride), s.x_stride, x_plane, 0};
        const Operand scaled{reinterpret_cast<const short *>(scaled_x + (int64_t)first * s.x_stride), s.x_stride, x_plane, 0};
        const int tokens = most > 0 ? most : 0;
        LogitsArgs l{w, kFull ? scaled : plain, pairs, s.width / kStepK, first, tokens, s.vocab, s.padded, head, row_target, target_logit,
                     reinterpret_cast<float2 *>(space + s.stats), s.groups, s.keep, space + s.kept, s.slope_stride, kFull ? x_exponents : nullptr,
                     kFull ? w_exponents : nullptr};
        RowsArgs r{first, tokens, s.vocab, s.padded, s.groups, kShapeSpan[s.logits_shape], head, row_of, row_target, target_logit,
                   reinterpret_cast<const float2 *>(space + s.stats), losses, s.keep, s.slope_planes, space + s.kept, space + s.slopes,
                   s.slope_stride, slope_plane, kFull ? w_exponents : nullptr, x_exponents, c.dw ? s.dw_slope_planes : 0,
                   reinterpret_cast<_Float16 *>(space + s.dw_slopes)};
        if (tokens > 0) {
            launch_logits<T>(s.logits_shape, l, tokens, stream);
            rows_kernel<T><<<(tokens + kStepK - 1) / kStepK * kStepK, kRowBlock, 0, stream>>>(r);
        }
        if (!s.gradients) continue;
        const Operand slopes{reinterpret_cast<const short *>(space + s.slopes), s.slope_stride, slope_plane, 0};
        if (c.dx && tokens > 0) {
            ProductArgs a{};
            a.p = w, a.p.rows = s.dim, a.q = slopes, a.pairs = pairs;
            a.first = first, a.most = tokens, a.steps = s.padded / kStepK, a.limit_p = s.vocab;
            a.splits = s.dx_splits, a.partial = reinterpret_cast<float *>(space + s.partial), a.partial_rows = tokens;
            a.head = head, a.row_of = row_of, a.unscale = kFull ? 1.0f : 1.0f / kSlopeScale<T>, a.exponent = kFull ? &head->w_exponent : nullptr;
            a.out = reinterpret_cast<void *>(c.dx), a.out_stride = c.dx_stride, a.out_type = c.data_type;
            a.out_aligned = c.dx % 16 == 0 && c.dx_stride * sizeof(I) % 16 == 0;
            launch_product<T, false>(s.dx_shape, a, s.dim, tokens, stream);
        }
        if (c.dw) {
            ProductArgs a{};
            const bool scales = s.dw_slope_planes != 0;
            a.p = scales ? scaled : plain, a.p.rows = s.dim;
            a.q = scales ? Operand{reinterpret_cast<const short *>(space + s.dw_slopes), s.slope_stride, slope_plane, 0} : slopes, a.q.rows = s.vocab;
            a.pairs = kFull ? kBothParts : scales || s.slope_planes == 2 ? kPartsOfQ : kOnePair;
            a.first = first, a.most = tokens, a.head = head, a.unscale = scales ? 1.0f : 1.0f / kSlopeScale<T>;
            a.exponent = scales ? &head->x_exponent : nullptr;
            a.splits = s.dw_splits, a.partial = reinterpret_cast<float *>(space + s.partial), a.partial_rows = s.vocab;
            const bool last = k + 1 == s.chunks;
            float *sums = reinterpret_cast<float *>(space + s.sums);
            if (s.sum_weights && !last) {
                a.out = sums, a.out_stride = s.dim, a.out_type = kFloat32, a.accumulate = k > 0;
                a.out_aligned = s.dim % 4 == 0;
            } else {
                a.out = reinterpret_cast<void *>(c.dw), a.out_stride = c.dw_stride, a.out_type = c.gradient_type;
                a.out_aligned = c.dw % 16 == 0 && c.dw_stride * type_bytes(c.gradient_type) % 16 == 0;
                a.accumulate = c.accumulate || (k > 0 && !s.sum_weights);
                a.add = s.sum_weights && k > 0 ? sums : nullptr;
            }
            a.skip_empty = a.accumulate && !a.add;
            if (scales) launch_product<_Float16, true>(s.dw_shape, a, s.dim, s.vocab, stream);
            else launch_product<T, true>(s.dw_shape, a, s.dim, s.vocab, stream);
        }
    }
    total_kernel<<<1, 1024, 0, stream>>>(losses, s.n, c.mean, head, reinterpret_cast<float *>(c.loss));
}

static bool loss_sizes(int n, int vocab, int dim, int data_type, int gradient_type)
{
    return n >= 0 && n <= 1 << 24 && vocab > 0 && vocab <= 1 << 22 && dim > 0 && dim <= 1 << 20 && (int64_t)vocab * dim <= kMostOutputs &&
           known_type(data_type) && (gradient_type == kFloat32 || gradient_type == data_type);
}

}  // namespace gm

using namespace gm;

extern "C" {

uintptr_t gm_linear_cross_entropy_workspace(int num_tokens, int vocab_size, int dim, uintptr_t weight_buffer, int weight_stride,
                                            int data_type, int gradient_type, int with_gradients)
{
    if (!loss_sizes(num_tokens, vocab_size, dim, data_type, gradient_type)) return 0;
    return loss_plan(num_tokens, vocab_size, dim, weights_fit(weight_buffer, dim, weight_stride, data_type), data_type, gradient_type,
                     with_gradients != 0, 0).bytes;
}

uintptr_t gm_linear_cross_entropy_least_workspace(int num_tokens, int vocab_size, int dim, uintptr_t weight_buffer, int weight_stride,
                                                  int data_type, int gradient_type, int with_gradients)
{
    if (!loss_sizes(num_tokens, vocab_size, dim, data_type, gradient_type)) return 0;
    LossPlan s;
    fitting_plan(s, 0, num_tokens, vocab_size, dim, weights_fit(weight_buffer, dim, weight_stride, data_type), data_type, gradient_type,
                 with_gradients != 0);
    return s.bytes;
}

int gm_linear_cross_entropy_plan(int num_tokens, int vocab_size, int dim, uintptr_t weight_buffer, int weight_stride, int data_type,
                                 int gradient_type, int with_gradients, uintptr_t workspace_bytes, int *plan)
{
    if (!plan) return kRcNil;
    if (!known_type(data_type) || (gradient_type != kFloat32 && gradient_type != data_type)) return kRcType;
    if (!loss_sizes(num_tokens, vocab_size, dim, data_type, gradient_type) || weight_stride < dim) return kRcRange;
    LossPlan s;
    if (!fitting_plan(s, workspace_bytes, num_tokens, vocab_size, dim, weights_fit(weight_buffer, dim, weight_stride, data_type), data_type,
                      gradient_type, with_gradients != 0))
        return kRcWorkspace;
    const int is[7] = {s.chunk, s.logits_shape, s.dx_shape, s.dx_splits, s.dw_shape, s.dw_splits, s.sum_weights};
    for (int k = 0; k < 7; k++) plan[k] = is[k];
    return 0;
}

int execute_linear_cross_entropy(uintptr_t device, uintptr_t command_queue, uintptr_t hidden_buffer, uintptr_t weight_buffer,
                                 uintptr_t target_buffer, uintptr_t losses_buffer, uintptr_t loss_buffer,
                                 uintptr_t hidden_gradient_buffer, uintptr_t weight_gradient_buffer, int num_tokens, int vocab_size,
                                 int dim, int hidden_stride, int weight_stride, int hidden_gradient_stride, int weight_gradient_stride,
                                 int data_type, int gradient_type, int ignore_index, int mean, float gradient_scale, uintptr_t amp_state,
                                 int accumulate, uintptr_t workspace, uintptr_t workspace_bytes)
try {
    clear_error();
    if (device == 0) return kRcDevice;
    if (hidden_buffer == 0 || weight_buffer == 0 || target_buffer == 0 || losses_buffer == 0 || loss_buffer == 0) return kRcNil;
    if (!known_type(data_type) || (gradient_type != kFloat32 && gradient_type != data_type)) return kRcType;
    const bool gradients = hidden_gradient_buffer != 0 || weight_gradient_buffer != 0;
    if (!loss_sizes(num_tokens, vocab_size, dim, data_type, gradient_type) || hidden_stride < dim || weight_stride < dim ||
        (hidden_gradient_buffer != 0 && hidden_gradient_stride < dim) || (weight_gradient_buffer != 0 && weight_gradient_stride < dim)) {
        set_error("sizes: %d tokens, vocabulary %d, dimension %d, strides %d, %d, %d and %d", num_tokens, vocab_size, dim, hidden_stride,
                  weight_stride, hidden_gradient_stride, weight_gradient_stride);
        return kRcRange;
    }
    const size_t in = type_bytes(data_type), out = type_bytes(gradient_type), n = (size_t)num_tokens, v = (size_t)vocab_size, d = (size_t)dim;
    if (!element_aligned("hidden", hidden_buffer, in) || !element_aligned("weight", weight_buffer, in) ||
        !element_aligned("targets", target_buffer, 4) || !element_aligned("losses", losses_buffer, 4) ||
        !element_aligned("loss", loss_buffer, 4) || !element_aligned("hidden gradient", hidden_gradient_buffer, in) ||
        !element_aligned("weight gradient", weight_gradient_buffer, out) ||
        !rows_fit("hidden", hidden_buffer, n, d, (size_t)hidden_stride, in) ||
        !rows_fit("weight", weight_buffer, v, d, (size_t)weight_stride, in) || !rows_fit("targets", target_buffer, 1, n, n, 4) ||
        !rows_fit("losses", losses_buffer, 1, n, n, 4) || !rows_fit("loss", loss_buffer, 1, 2, 2, 4) ||
        (hidden_gradient_buffer && !rows_fit("hidden gradient", hidden_gradient_buffer, n, d, (size_t)hidden_gradient_stride, in)) ||
        (weight_gradient_buffer && !rows_fit("weight gradient", weight_gradient_buffer, v, d, (size_t)weight_gradient_stride, out)))
        return kRcRange;
    LossPlan plan;
    if (!fitting_plan(plan, workspace ? (size_t)workspace_bytes : 0, num_tokens, vocab_size, dim,
                      weights_fit(weight_buffer, dim, weight_stride, data_type), data_type, gradient_type, gradients) ||
        workspace % 256 != 0 || !rows_fit("workspace", workspace, 1, plan.bytes, plan.bytes, 1)) {
        set_error("the workspace holds %zu bytes (or is not aligned to 256): at least %zu are needed", (size_t)workspace_bytes, plan.bytes);
        return kRcWorkspace;
    }
    Context *ctx = resolve_device(device);
    if (!ctx) return kRcNoGpu;
    hipStream_t stream;
    if (!queue_stream(ctx, command_queue, &stream)) return kRcQueue;
    LossCall c{hidden_buffer, weight_buffer, target_buffer, losses_buffer, loss_buffer, hidden_gradient_buffer, weight_gradient_buffer,
               hidden_stride, weight_stride, hidden_gradient_stride, weight_gradient_stride, data_type, gradient_type, ignore_index,
               mean != 0, accumulate != 0, gradient_scale, AmpScaleView{}, reinterpret_cast<char *>(workspace)};
    if (amp_state != 0 && !amp_scale_view(amp_state, ctx, &c.amp)) return kRcAmp;
    DeviceScope scope(ctx);
    if (!scope.ok()) return kRcHip;
    if (data_type == kFloat32) launch_loss<float, _Float16>(c, plan, stream);
    else if (data_type == kFloat16) launch_loss<_Float16, _Float16>(c, plan, stream);
    else launch_loss<__bf16, __bf16>(c, plan, stream);
    return hip_ok(hipGetLastError(), "linear cross entropy launch") ? 0 : kRcHip;
} catch (...) {
    note_exception();
    return kRcHip;
}

}  // extern "C"
