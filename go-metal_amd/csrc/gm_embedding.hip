// Embedding lookup with scaling (and the embedding's dropout), and its gradient by sorted tokens.
//
// Gradient: G[v] (+)= scale * sum over the positions i with token v, in the order of i, of dy[i].  The tokens are
// sorted (stably: equal tokens keep their positions' order), so that each row of the table is one run of the sorted
// list; runs are summed in fp32 registers and each row is written once.  No atomics: the order of every sum is
// fixed by the tokens alone, and results repeat bit for bit.
#include "gm_ops.hpp"

#include "../../include/gometal_hip.h"

namespace gm {

constexpr int kLookupBlock = 256;

// One lane moves eight elements (16 bytes of a 16-bit type); lanes run over the rows' vectors without gaps, so short
// rows share a workgroup.  Memory bounds it: 8192 rows of 4096 bf16, dropped out, 23 us = 5.9 TB/s of reads and writes, some
// rows from the caches.  A single row is one launch's latency, 2.5 us on the device.  A token outside the vocabulary is padding and gives a row of zeros.
template <typename T>
__global__ void __launch_bounds__(kLookupBlock)
lookup_kernel(const T *table, const int *tokens, T *out, uint64_t first, uint32_t rows, uint32_t vocab, uint32_t dim, uint32_t per_row,
              int64_t table_stride, int64_t out_stride, float scale, DropoutParams d, bool aligned)
{
    const uint64_t base = (uint64_t)blockIdx.x * kLookupBlock;
    const uint32_t base_row = (uint32_t)(base / per_row), base_vec = (uint32_t)(base - (uint64_t)base_row * per_row);
    const uint32_t step = (base_vec + threadIdx.x) / per_row;
    const uint32_t row = base_row + step, col = (base_vec + threadIdx.x - step * per_row) * 8;
    if (row >= rows) return;
    const int count = dim - col < 8 ? (int)(dim - col) : 8;
    const bool whole = aligned && count == 8;
    const uint32_t token = (uint32_t)tokens[row];
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (token < vocab) {
        load8(table + (int64_t)token * table_stride + col, whole, count, v);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = v[e] * scale;
        if (d.state) {
            const DropoutState st = *d.state;
            drop8(v, first + (uint64_t)row * dim + col, d, st);      // first: the launch's first element
        }
    }
    store8(out + (int64_t)row * out_stride + col, whole, count, v);
}

// ---------------------------------------------------------------------------------------- sorting the tokens ----
// A list of up to kSortChunk tokens is sorted by counting: a token's place is the number of tokens before it in the
// order (token, position).  That is n^2 comparisons without a single dependent pass: 8192 tokens are 67M
// comparisons over the whole chip, 9.7 us; the vector units' issue bounds it.  Longer lists are sorted in chunks; a
// token's place in the whole is then its place in its chunk plus a binary search in every other one.  Comparisons grow with
// the chunk and searches with the number of chunks: 32768 tokens take 27 + 10 us in chunks of 8192 and 9.5 + 11 us in
// chunks of 2048, so those are taken as long as a token's searches are no more than two a lane of the merge.
constexpr int kSortChunk = 8192, kShortChunk = 2048;
constexpr int kMergeLanes = 16;      // lanes that share an element's searches
constexpr int kShortChunks = 2 * kMergeLanes * kShortChunk;      // the longest list in short chunks
constexpr int kMostTokens = 1 << 22;      // the merge's searches grow with the square of the list: 512 chunks are enough of them
constexpr int kSortLanes = 16;        // lanes that share a part of the chunk; each compares kSortOwn tokens of its own with it
constexpr int kSortOwn = 2;
constexpr int kSortRows = kSortLanes * kSortOwn, kSortSlices = 64, kSortBlock = kSortLanes * kSortSlices;
constexpr uint32_t kNoToken = 0xFFFFFFFFu;
// Vocabularies below this fit a sort key of token and position in one 32-bit word, one comparison instead of three.
constexpr uint32_t kShortVocab = (1u << 19) - 1;

// SHORT: a key is token << 13 | position in the chunk; otherwise the token, and positions are compared where tokens are equal.
template <bool SHORT, int CHUNK>
__global__ void __launch_bounds__(kSortBlock)
sort_chunk_kernel(const int *tokens, uint32_t n, uint32_t vocab, int padding, uint32_t *keys, uint32_t *positions)
{
    __shared__ __attribute__((aligned(16))) uint32_t all[CHUNK];
    __shared__ uint32_t before[kSortRows];
    constexpr uint32_t kBlocks = CHUNK / kSortRows;      // per chunk
    const uint32_t chunk = blockIdx.x / kBlocks, first = chunk * CHUNK, row = (blockIdx.x - chunk * kBlocks) * kSortRows;
    const uint32_t len = n - first < CHUNK ? n - first : CHUNK;
    if (row >= len) return;
    const uint32_t filled = (len + 4 * kSortSlices - 1) / (4 * kSortSlices) * (4 * kSortSlices);      // whole rounds of fours
    // Padding and tokens outside the vocabulary sort behind everything else; what fills the last round, behind them.
    for (uint32_t i = threadIdx.x; i < filled; i += kSortBlock) {
        const int t = i < len ? tokens[first + i] : -1;
        const bool counts = (uint32_t)t < vocab && t != padding;
        all[i] = SHORT ? (i < len ? (counts ? (uint32_t)t : kShortVocab) << 13 | i : kNoToken) : counts ? (uint32_t)t : kNoToken;
    }
    if (threadIdx.x < kSortRows) before[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t lane = threadIdx.x % kSortLanes, slice = threadIdx.x / kSortLanes;
    uint32_t mine[kSortOwn], key[kSortOwn], count[kSortOwn];
#pragma unroll
    for (int o = 0; o < kSortOwn; o++) {
        mine[o] = row + o * kSortLanes + lane;
        key[o] = mine[o] < len ? all[mine[o]] : kNoToken;
        count[o] = 0;
    }
    for (uint32_t j = slice * 4; j < filled; j += 4 * kSortSlices) {      // (a wavefront's four parts lie side by side)
        const uint4 k4 = *reinterpret_cast<const uint4 *>(&all[j]);
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int o = 0; o < kSortOwn; o++)
#pragma unroll
            for (uint32_t c = 0; c < 4; c++)
                count[o] += SHORT ? k[c] < key[o] : (uint32_t)((k[c] < key[o]) | ((k[c] == key[o]) & (j + c < mine[o])));
    }
#pragma unroll
    for (int o = 0; o < kSortOwn; o++) atomicAdd(&before[o * kSortLanes + lane], count[o]);      // whole numbers: their order does not matter
    __syncthreads();
    const uint32_t me = row + threadIdx.x;
    if (threadIdx.x < kSortRows && me < len) {
        const uint32_t token = SHORT ? all[me] >> 13 : all[me];
        keys[first + before[threadIdx.x]] = SHORT && token == kShortVocab ? kNoToken : token;
        positions[first + before[threadIdx.x]] = first + me;
    }
}

// How many of a sorted list's keys are below `key` (or, with `through`, not above it).
__device__ inline uint32_t keys_before(const uint32_t *keys, uint32_t n, uint32_t key, bool through)
{
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        const uint32_t k = keys[mid];
        if (k < key || (through && k == key)) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Sixteen lanes an element, a chunk each at a time: a search's loads depend on each other, the lanes' do not.  11 us for 32768
// tokens, the latency of eleven loads behind one another.
__global__ void __launch_bounds__(256)
merge_chunks_kernel(const uint32_t *keys, const uint32_t *positions, uint32_t n, uint32_t chunk, uint32_t *out_keys, uint32_t *out_positions)
{
    const uint32_t i = blockIdx.x * (256 / kMergeLanes) + threadIdx.x / kMergeLanes, lane = threadIdx.x % kMergeLanes;
    if (i >= n) return;
    const uint32_t key = keys[i], mine = i / chunk;
    uint32_t place = lane == 0 ? i - mine * chunk : 0;
    for (uint32_t c = lane; c * chunk < n; c += kMergeLanes) {
        if (c == mine) continue;
        const uint32_t first = c * chunk, len = n - first < chunk ? n - first : chunk;
        place += keys_before(keys + first, len, key, c < mine);      // equal tokens of earlier chunks come first
    }
#pragma unroll
    for (int o = kMergeLanes / 2; o; o >>= 1) place += __shfl_xor(place, o);
    if (lane == 0) {
        out_keys[place] = key;
        out_positions[place] = positions[i];
    }
}

// ------------------------------------------------------------------------------------------ summing the runs ----
// The sorted list is cut into pieces of 8 to 32 entries, so that a token that fills a tenth of a batch is summed by
// many workgroups.  A run that lies in one piece goes straight to its row; of one that crosses a border every piece
// leaves a partial sum (slot 0: the run the piece begins in the middle of; slot 1: the run it ends in the middle
// of), which join_runs_kernel adds up in the pieces' order.  Memory bounds the sums and the fill beside them: 131072 x 2048
// fp32 from 32768 rows of bf16, 1.21 GB, 220 us = 5.5 TB/s; the joins take 6 to 10 us, latency.
constexpr int kSumBlock = 64;              // one wavefront, eight elements a lane

// Long pieces leave fewer partial sums, short ones more wavefronts: the longest that leave four for each SIMD.
static uint32_t piece_for(size_t n, size_t dim)
{
    const size_t tiles = (dim + kSumBlock * 8 - 1) / (kSumBlock * 8);
    return n * tiles >= 4096 * 32 ? 32 : n * tiles >= 4096 * 16 ? 16 : 8;
}

struct SumArgs {
    const uint32_t *keys, *positions;
    uint32_t n, dim;
    int64_t dy_stride, out_stride;
    float scale;
    int accumulate;
    float *partial;                        // [piece][2][dim]
    DropoutParams d;
    bool in_aligned, out_aligned;
    uint32_t col_tiles, piece, sum_blocks;
};

// Rows that no token names are written with zeros by the workgroups behind the summing ones: a wavefront takes rows of 16 KiB
// together, up to 64, and each of its lanes looks one of them up in the sorted list.  The store is most of a gradient's
// time, and the sums' reads run beside it.
struct FillArgs {
    char *out;
    int64_t row_bytes, stride_bytes;
    uint32_t rows, rows_each;       // rows of one workgroup
};

__device__ inline void fill_rows(const FillArgs &f, const uint32_t *keys, uint32_t n, uint32_t block)
{
    typedef uint32_t Vec __attribute__((ext_vector_type(4)));
    const uint32_t first = block * f.rows_each, count = f.rows - first < f.rows_each ? f.rows - first : f.rows_each, lane = threadIdx.x;
    bool named = false;
    if (lane < count) {
        const uint32_t at = keys_before(keys, n, first + lane, false);
        named = at < n && keys[at] == first + lane;
    }
    const uint64_t skip = __ballot(named);
    for (uint32_t r = 0; r < count; r++) {
        if (skip >> r & 1) continue;
        char *to = f.out + (int64_t)(first + r) * f.stride_bytes;
        int64_t head = (int64_t)((16 - ((uintptr_t)to & 15)) & 15);
        head = head < f.row_bytes ? head : f.row_bytes;
        const uint32_t whole = (uint32_t)((f.row_bytes - head) / 16);
        // (past the caches: the rows are not read again, and what the sums read stays there: 86 -> 73 us)
        for (uint32_t i = lane; i < whole; i += kSumBlock) __builtin_nontemporal_store(Vec{0u, 0u, 0u, 0u}, reinterpret_cast<Vec *>(to + head) + i);
        if (lane < 32) {         // (elements are 2 or 4 bytes: heads and tails are pairs of bytes)
            const int64_t at = lane < 8 ? (int64_t)lane * 2 : head + (int64_t)whole * 16 + ((int64_t)lane - 8) * 2, end = lane < 8 ? head : f.row_bytes;
            if (at < end) *reinterpret_cast<uint16_t *>(to + at) = 0;
        }
    }
}

// Eight elements of a row that are there already.
template <typename O>
__device__ inline void read_row(const O *out, const SumArgs &a, uint32_t row, uint32_t col, int count, float (&old)[8])
{
    load8(out + (int64_t)row * a.out_stride + col, a.out_aligned && count == 8, count, old);
}

template <typename O>
__device__ inline void write_row(O *out, const SumArgs &a, uint32_t row, uint32_t col, int count, const float (&acc)[8], const float (&old)[8])
{
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        v[e] = acc[e] * a.scale;
        if (a.accumulate) v[e] = old[e] + v[e];
    }
    store8(out + (int64_t)row * a.out_stride + col, a.out_aligned && count == 8, count, v);
}

// ADD: the sums are added to the rows, whose old values are loaded beside the gradients' rows (loaded behind each sum, where a
// wavefront waits for them row by row: 4097 rows into 50001 x 1000 fp32 21.4 us a call instead of 20.5).
template <typename T, typename O, bool ADD>
__global__ void __launch_bounds__(kSumBlock)
sum_runs_kernel(const T *dy, O *out, SumArgs a, FillArgs fill)
{
    if (blockIdx.x >= a.sum_blocks) {
        fill_rows(fill, a.keys, a.n, blockIdx.x - a.sum_blocks);
        return;
    }
    const uint32_t piece = blockIdx.x / a.col_tiles;
    const uint32_t col = (blockIdx.x - piece * a.col_tiles) * (kSumBlock * 8) + threadIdx.x * 8;
    const uint32_t lo = piece * a.piece, hi = a.n - lo < a.piece ? a.n : lo + a.piece;
    // the piece's entries, one a lane: later every lane takes them from there
    const uint32_t l = threadIdx.x;
    const uint32_t my_key = lo + l < hi ? a.keys[lo + l] : 0xFFFFFFFFu;
    const uint32_t my_pos = lo + l < hi ? a.positions[lo + l] : 0u;
    const uint32_t key_before = lo > 0 ? a.keys[lo - 1] : 0xFFFFFFFFu;
    const uint32_t key_after = hi < a.n ? a.keys[hi] : 0xFFFFFFFFu;
    const uint32_t entries = (uint32_t)__popcll(__ballot(my_key != 0xFFFFFFFFu));      // padding is sorted to the end
    if (entries == 0) return;
    // (lanes behind the last column stay: the others read their entries)
    const int count = col >= a.dim ? 0 : a.dim - col < 8 ? (int)(a.dim - col) : 8;
    const bool whole = a.in_aligned && count == 8;
    DropoutState st = {};
    if (a.d.state) st = *a.d.state;
    float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    bool from_before = __builtin_amdgcn_readlane(my_key, 0) == key_before;
    constexpr uint32_t kAhead = sizeof(T) == 2 && !ADD ? 8 : 4;         // rows in flight a lane
    const auto key_behind = [&](uint32_t at) {
        return at + 1 < entries ? (uint32_t)__builtin_amdgcn_readlane(my_key, at + 1) : lo + entries == hi ? key_after : 0xFFFFFFFFu;
    };
    for (uint32_t i = 0; i < entries; i += kAhead) {
        float v[kAhead][8];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const uint32_t at = i + k < entries ? i + k : entries - 1;
            load8(dy + (int64_t)(uint32_t)__builtin_amdgcn_readlane(my_pos, at) * a.dy_stride + col, whole, count, v[k]);
        }
        float old[kAhead][8];
        if (ADD) {
#pragma unroll
            for (uint32_t k = 0; k < kAhead; k++) {
                const uint32_t at = i + k < entries ? i + k : entries - 1, key = __builtin_amdgcn_readlane(my_key, at);
                if (key_behind(at) != key) read_row(out, a, key, col, count, old[k]);      // a run ends here
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            if (i + k >= entries) break;
            const uint32_t at = i + k;
            const uint32_t key = __builtin_amdgcn_readlane(my_key, at);
            if (a.d.state) drop8(v[k], (uint64_t)(uint32_t)__builtin_amdgcn_readlane(my_pos, at) * a.dim + col, a.d, st);
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = acc[e] + v[k][e];
            const bool last = at + 1 == entries;
            const bool goes_on = key_behind(at) == key;
            if (goes_on && !last) continue;        // (the last entry of a piece leaves its unfinished run behind)
            if (from_before || goes_on) {
                store8(a.partial + ((int64_t)piece * 2 + (from_before ? 0 : 1)) * a.dim + col, count == 8 && a.dim % 4 == 0, count, acc);
            } else if (count > 0) {
                write_row(out, a, key, col, count, acc, old[k]);
            }
            from_before = false;
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = 0.0f;
        }
    }
}

// A run that begins in piece c and goes on behind it: its partial sums, added up in the pieces' order.
template <typename O>
__global__ void __launch_bounds__(kSumBlock)
join_runs_kernel(O *out, SumArgs a)
{
    const uint32_t piece = blockIdx.x / a.col_tiles;
    const uint32_t col = (blockIdx.x - piece * a.col_tiles) * (kSumBlock * 8) + threadIdx.x * 8;
    const uint32_t border = (piece + 1) * a.piece;      // (the grid leaves the last piece out: border < n)
    const uint32_t key = a.keys[border - 1];
    if (key == 0xFFFFFFFFu || a.keys[border] != key) return;
    const uint32_t lo = piece * a.piece;
    if (lo > 0 && a.keys[lo - 1] == key) return;       // it began in an earlier piece
    // the pieces it goes into: those whose first key is this one, 64 looked at together (all lanes, also those behind the last column)
    uint32_t last = piece + 1;
    for (uint32_t more = 64; more == 64; last += more) {
        const uint32_t first = (last + 1 + threadIdx.x) * a.piece;
        const uint64_t others = ~__ballot(first < a.n && a.keys[first] == key);
        more = others ? (uint32_t)__builtin_ctzll(others) : 64;
    }
    if (col >= a.dim) return;
    const int count = a.dim - col < 8 ? (int)(a.dim - col) : 8;
    const bool whole = count == 8 && a.dim % 4 == 0;
    float acc[8], old[8];
    if (a.accumulate) read_row(out, a, key, col, count, old);
    load8(a.partial + ((int64_t)piece * 2 + 1) * a.dim + col, whole, count, acc);
    constexpr uint32_t kAhead = 8;      // partial sums in flight a lane (a word that fills a tenth of a batch has a hundred)
    for (uint32_t c = piece + 1; c <= last; c += kAhead) {
        float v[kAhead][8];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) load8(a.partial + (int64_t)(c + k <= last ? c + k : last) * 2 * a.dim + col, whole, count, v[k]);
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++)
            if (c + k <= last) {
#pragma unroll
                for (int e = 0; e < 8; e++) acc[e] = acc[e] + v[k][e];
            }
    }
    write_row(out, a, key, col, count, acc, old);
}

// ------------------------------------------------------------------------------------------------- host side ----
struct GradientSpace {
    size_t keys, positions, chunk_keys, chunk_positions, partial, bytes;
};

static GradientSpace gradient_space(size_t n, size_t dim)
{
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    GradientSpace s;
    size_t at = 0;
    s.keys = at, at += up(4 * n);
    s.positions = at, at += up(4 * n);
    s.chunk_keys = at, at += n > kSortChunk ? up(4 * n) : 0;
    s.chunk_positions = at, at += n > kSortChunk ? up(4 * n) : 0;
    const size_t piece = piece_for(n, dim);
    s.partial = at, at += n > piece ? up((n + piece - 1) / piece * 2 * dim * 4) : 0;
    s.bytes = at;
    return s;
}

template <typename T, typename O>
static void launch_sums(const SumArgs &a, const FillArgs &fill, uintptr_t dy, uintptr_t out, uint32_t fills, uint32_t join_grid, hipStream_t stream)
{
    if (a.sum_blocks + fills)
        (a.accumulate ? sum_runs_kernel<T, O, true> : sum_runs_kernel<T, O, false>)<<<a.sum_blocks + fills, kSumBlock, 0, stream>>>(
            reinterpret_cast<const T *>(dy), reinterpret_cast<O *>(out), a, fill);
    if (join_grid) join_runs_kernel<O><<<join_grid, kSumBlock, 0, stream>>>(reinterpret_cast<O *>(out), a);
}

template <typename T>
static void launch_lookup(uintptr_t table, uintptr_t tokens, uintptr_t out, int n, int vocab, int dim, int table_stride,
                          int out_stride, float scale, const DropoutParams &d, hipStream_t stream)
{
    const bool aligned = (table | out) % 16 == 0 && (size_t)table_stride * sizeof(T) % 16 == 0 && (size_t)out_stride * sizeof(T) % 16 == 0;
    const uint32_t per_row = ((uint32_t)dim + 7) / 8;
    // (a launch can address fewer than 2^32 lanes: more vectors than 2^31 go in parts of whole rows)
    const uint32_t rows_each = (1u << 31) / per_row;
    for (uint32_t first = 0; first < (uint32_t)n; first += rows_each) {
        const uint32_t rows = (uint32_t)n - first < rows_each ? (uint32_t)n - first : rows_each;
        const uint32_t grid = (uint32_t)(((uint64_t)rows * per_row + kLookupBlock - 1) / kLookupBlock);
        lookup_kernel<T><<<grid, kLookupBlock, 0, stream>>>(reinterpret_cast<const T *>(table), reinterpret_cast<const int *>(tokens) + first,
                                                            reinterpret_cast<T *>(out) + (int64_t)first * out_stride, (uint64_t)first * (uint32_t)dim, rows,
                                                            (uint32_t)vocab, (uint32_t)dim, per_row, table_stride, out_stride, scale, d, aligned);
    }
}

// What the two entry points check alike.
static int embedding_arguments(uintptr_t tokens, uintptr_t rng_state, int n, int vocab, int dim, int stride_a, int stride_b,
                               float probability, int site, DropoutParams *d)
{
    if (n < 0 || vocab <= 0 || dim <= 0 || stride_a < dim || stride_b < dim) {
        set_error("sizes: %d tokens, vocabulary %d, dimension %d, strides %d and %d", n, vocab, dim, stride_a, stride_b);
        return kRcRange;
    }
    if (!dropout_params(probability, rng_state, site, d)) return kRcRange;
    if (rng_state == 0 && probability > 0.0f) return kRcNil;
    if (!element_aligned("tokens", tokens, 4) || !element_aligned("generator state", rng_state, 16) ||
        !rows_fit("tokens", tokens, 1, (size_t)n, (size_t)n, 4) || !rows_fit("generator state", rng_state, 1, 4, 4, 4))
        return kRcRange;
    return 0;
}

}  // namespace gm

using namespace gm;

extern "C" {

int execute_embedding_lookup(uintptr_t device, uintptr_t command_queue, uintptr_t table_buffer, uintptr_t token_buffer,
                             uintptr_t output_buffer, int num_tokens, int vocab_size, int dim, int table_stride, int output_stride,
                             int data_type, float scale, float dropout_probability, uintptr_t rng_state, int dropout_site)
try {
    clear_error();
    if (device == 0) return kRcDevice;
    if (table_buffer == 0 || token_buffer == 0 || output_buffer == 0) return kRcNil;
    if (!known_type(data_type)) return kRcType;
    DropoutParams d;
    if (int rc = embedding_arguments(token_buffer, rng_state, num_tokens, vocab_size, dim, table_stride, output_stride,
                                     dropout_probability, dropout_site, &d))
        return rc;
    const size_t element = type_bytes(data_type);
    if (!element_aligned("table", table_buffer, element) || !element_aligned("output", output_buffer, element) ||
        !rows_fit("table", table_buffer, (size_t)vocab_size, (size_t)dim, (size_t)table_stride, element) ||
        !rows_fit("output", output_buffer, (size_t)num_tokens, (size_t)dim, (size_t)output_stride, element))
        return kRcRange;
    if ((uint64_t)num_tokens * (((uint32_t)dim + 7) / 8) > 1ull << 39) {
        set_error("a lookup of %d rows of %d elements: at most 2^39 groups of eight elements", num_tokens, dim);
        return kRcRange;
    }
    Context *ctx = resolve_device(device);
    if (!ctx) return kRcNoGpu;
    hipStream_t stream;
    if (!queue_stream(ctx, command_queue, &stream)) return kRcQueue;
    if (num_tokens == 0) return 0;
    DeviceScope scope(ctx);
    if (!scope.ok()) return kRcHip;
    const auto launch = data_type == kFloat32 ? launch_lookup<float> : data_type == kFloat16 ? launch_lookup<_Float16> : launch_lookup<__bf16>;
    launch(table_buffer, token_buffer, output_buffer, num_tokens, vocab_size, dim, table_stride, output_stride, scale, d, stream);
    return hip_ok(hipGetLastError(), "embedding lookup launch") ? 0 : kRcHip;
} catch (...) {
    note_exception();
    return kRcHip;
}

uintptr_t gm_embedding_gradient_workspace(int num_tokens, int vocab_size, int dim)
{
    if (num_tokens < 0 || num_tokens > kMostTokens || vocab_size <= 0 || dim <= 0) return 0;
    return gradient_space((size_t)num_tokens, (size_t)dim).bytes;
}

int execute_embedding_gradient(uintptr_t device, uintptr_t command_queue, uintptr_t output_gradient_buffer, uintptr_t token_buffer,
                               uintptr_t table_gradient_buffer, int num_tokens, int vocab_size, int dim, int output_gradient_stride,
                               int table_gradient_stride, int data_type, int gradient_type, float scale, int padding_token,
                               int accumulate, float dropout_probability, uintptr_t rng_state, int dropout_site, uintptr_t workspace,
                               uintptr_t workspace_bytes)
try {
    clear_error();
    if (device == 0) return kRcDevice;
    if (output_gradient_buffer == 0 || token_buffer == 0 || table_gradient_buffer == 0) return kRcNil;
    if (!known_type(data_type) || (gradient_type != kFloat32 && gradient_type != data_type)) return kRcType;
    DropoutParams d;
    if (int rc = embedding_arguments(token_buffer, rng_state, num_tokens, vocab_size, dim, output_gradient_stride,
                                     table_gradient_stride, dropout_probability, dropout_site, &d))
        return rc;
    if (num_tokens > kMostTokens) {
        set_error("a gradient of %d tokens: at most %d at a time (accumulate the parts)", num_tokens, kMostTokens);
        return kRcRange;
    }
    const size_t in = type_bytes(data_type), out = type_bytes(gradient_type);
    if (!element_aligned("output gradient", output_gradient_buffer, in) || !element_aligned("table gradient", table_gradient_buffer, out) ||
        !rows_fit("output gradient", output_gradient_buffer, (size_t)num_tokens, (size_t)dim, (size_t)output_gradient_stride, in) ||
        !rows_fit("table gradient", table_gradient_buffer, (size_t)vocab_size, (size_t)dim, (size_t)table_gradient_stride, out))
        return kRcRange;
    const GradientSpace space = gradient_space((size_t)num_tokens, (size_t)dim);
    if (space.bytes > 0 && (workspace == 0 || workspace % 256 != 0 || workspace_bytes < space.bytes ||
                            !rows_fit("workspace", workspace, 1, space.bytes, space.bytes, 1))) {
        set_error("the workspace holds %zu bytes (or is not aligned to 256): %zu are needed", (size_t)workspace_bytes, space.bytes);
        return kRcWorkspace;
    }
    const uint32_t n = (uint32_t)num_tokens;
    SumArgs a{};
    a.col_tiles = ((uint32_t)dim + kSumBlock * 8 - 1) / (kSumBlock * 8);
    a.piece = piece_for(n, (size_t)dim);
    const uint64_t pieces = ((uint64_t)n + a.piece - 1) / a.piece;
    FillArgs fill{reinterpret_cast<char *>(table_gradient_buffer), (int64_t)dim * (int64_t)out, (int64_t)table_gradient_stride * (int64_t)out,
                  (uint32_t)vocab_size, 1};
    fill.rows_each = fill.row_bytes * 64 <= 16384 ? 64 : fill.row_bytes < 16384 ? (uint32_t)(16384 / fill.row_bytes) : 1;
    const uint64_t fills = accumulate ? 0 : ((uint64_t)vocab_size + fill.rows_each - 1) / fill.rows_each;
    if ((pieces * a.col_tiles + fills) * kSumBlock > 0xFFFFFFFFull) {
        set_error("a gradient of %d rows of %d elements, vocabulary %d, needs more lanes than one launch can address", num_tokens, dim, vocab_size);
        return kRcRange;
    }
    Context *ctx = resolve_device(device);
    if (!ctx) return kRcNoGpu;
    hipStream_t stream;
    if (!queue_stream(ctx, command_queue, &stream)) return kRcQueue;
    DeviceScope scope(ctx);
    if (!scope.ok()) return kRcHip;
    uint32_t *keys = reinterpret_cast<uint32_t *>(workspace + space.keys);
    uint32_t *positions = reinterpret_cast<uint32_t *>(workspace + space.positions);
    const bool chunks = n > kSortChunk;
    const uint32_t chunk = chunks && n <= kShortChunks ? kShortChunk : kSortChunk;
    uint32_t *to_keys = chunks ? reinterpret_cast<uint32_t *>(workspace + space.chunk_keys) : keys;
    uint32_t *to_positions = chunks ? reinterpret_cast<uint32_t *>(workspace + space.chunk_positions) : positions;
    if (n > 0) {
        // (of a list shorter than a chunk only the workgroups that have rows to place are launched)
        const uint32_t grid = chunks ? (n + chunk - 1) / chunk * (chunk / kSortRows) : (n + kSortRows - 1) / kSortRows;
        const bool word = (uint32_t)vocab_size < kShortVocab;
        const auto sort = chunk == kSortChunk ? (word ? sort_chunk_kernel<true, kSortChunk> : sort_chunk_kernel<false, kSortChunk>)
                                              : (word ? sort_chunk_kernel<true, kShortChunk> : sort_chunk_kernel<false, kShortChunk>);
        sort<<<grid, kSortBlock, 0, stream>>>(reinterpret_cast<const int *>(token_buffer), n, (uint32_t)vocab_size, padding_token, to_keys,
                                              to_positions);
    }
    if (chunks)
        merge_chunks_kernel<<<(n + 256 / kMergeLanes - 1) / (256 / kMergeLanes), 256, 0, stream>>>(to_keys, to_positions, n, chunk, keys, positions);
    a.keys = keys;
    a.positions = positions;
    a.n = n;
    a.dim = (uint32_t)dim;
    a.dy_stride = output_gradient_stride;
    a.out_stride = table_gradient_stride;
    a.scale = scale;
    a.accumulate = accumulate != 0;
    a.partial = reinterpret_cast<float *>(workspace + space.partial);
    a.d = d;
    a.in_aligned = output_gradient_buffer % 16 == 0 && (size_t)output_gradient_stride * in % 16 == 0;
    a.out_aligned = table_gradient_buffer % 16 == 0 && (size_t)table_gradient_stride * out % 16 == 0;
    a.sum_blocks = (uint32_t)(pieces * a.col_tiles);
    const uint32_t join_grid = pieces > 1 ? (uint32_t)(pieces - 1) * a.col_tiles : 0;
    const auto launch = data_type == kFloat32                                       ? launch_sums<float, float>
                        : data_type == kFloat16 && gradient_type == kFloat16        ? launch_sums<_Float16, _Float16>
                        : data_type == kFloat16                                     ? launch_sums<_Float16, float>
                        : gradient_type == kBFloat16                                ? launch_sums<__bf16, __bf16>
                                                                                    : launch_sums<__bf16, float>;
    launch(a, fill, output_gradient_buffer, table_gradient_buffer, (uint32_t)fills, join_grid, stream);
    return hip_ok(hipGetLastError(), "embedding gradient launch") ? 0 : kRcHip;
} catch (...) {
    note_exception();
    return kRcHip;
}

}  // extern "C"
