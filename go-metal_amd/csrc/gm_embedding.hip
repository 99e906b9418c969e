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
// rows share a workgroup.  A token outside the vocabulary is padding and gives a row of zeros.
template <typename T>
__global__ void __launch_bounds__(kLookupBlock)
lookup_kernel(const T *table, const int *tokens, T *out, uint32_t rows, uint32_t vocab, uint32_t dim, uint32_t per_row,
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
            drop8(v, (uint64_t)row * dim + col, d, st);
        }
    }
    store8(out + (int64_t)row * out_stride + col, whole, count, v);
}

// ---------------------------------------------------------------------------------------- sorting the tokens ----
// A list of up to kSortChunk tokens is sorted by counting: a token's place is the number of tokens before it in the
// order (token, position).  That is n^2 comparisons without a single dependent pass: 8192 tokens are 67M
// comparisons over the whole chip.  Longer lists are sorted in chunks; a token's place in the whole is then its
// place in its chunk plus a binary search in every other one.
constexpr int kSortChunk = 8192;
constexpr int kSortRows = 32;         // tokens a workgroup places
constexpr int kSortSlices = 32;       // parts of the chunk that its lanes compare with

// Padding and tokens outside the vocabulary sort behind everything else.
__device__ inline uint32_t sort_key(int token, uint32_t vocab, int padding)
{
    return (uint32_t)token < vocab && token != padding ? (uint32_t)token : 0xFFFFFFFFu;
}

__global__ void __launch_bounds__(kSortRows *kSortSlices)
sort_chunk_kernel(const int *tokens, uint32_t n, uint32_t vocab, int padding, uint32_t *keys, uint32_t *positions)
{
    __shared__ uint32_t all[kSortChunk];
    __shared__ uint32_t before[kSortRows];
    const uint32_t first = blockIdx.y * kSortChunk;
    const uint32_t len = n - first < kSortChunk ? n - first : kSortChunk;
    if (blockIdx.x * kSortRows >= len) return;
    const uint32_t filled = (len + 4 * kSortSlices - 1) / (4 * kSortSlices) * (4 * kSortSlices);      // whole slices of fours
    for (uint32_t i = threadIdx.x; i < filled; i += kSortRows * kSortSlices)
        all[i] = i < len ? sort_key(tokens[first + i], vocab, padding) : 0xFFFFFFFFu;
    if (threadIdx.x < kSortRows) before[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t r = threadIdx.x % kSortRows, slice = threadIdx.x / kSortRows;
    const uint32_t mine = blockIdx.x * kSortRows + r;
    const uint32_t key = mine < len ? all[mine] : 0xFFFFFFFFu;
    const uint32_t per = filled / kSortSlices;
    uint32_t count = 0;
    for (uint32_t j = slice * per; j < (slice + 1) * per; j += 4) {
        const uint4 k = *reinterpret_cast<const uint4 *>(&all[j]);
        // (the filling behind the list has the largest key and later positions: it is never before anything)
        count += (k.x < key) | ((k.x == key) & (j < mine));
        count += (k.y < key) | ((k.y == key) & (j + 1 < mine));
        count += (k.z < key) | ((k.z == key) & (j + 2 < mine));
        count += (k.w < key) | ((k.w == key) & (j + 3 < mine));
    }
    atomicAdd(&before[r], count);      // whole numbers: their order does not matter
    __syncthreads();
    if (threadIdx.x < kSortRows && mine < len) {
        keys[first + before[r]] = key;
        positions[first + before[r]] = first + mine;
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

__global__ void __launch_bounds__(256)
merge_chunks_kernel(const uint32_t *keys, const uint32_t *positions, uint32_t n, uint32_t *out_keys, uint32_t *out_positions)
{
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t key = keys[i], mine = i / kSortChunk;
    uint32_t place = i % kSortChunk;
    for (uint32_t c = 0; c * kSortChunk < n; c++) {
        if (c == mine) continue;
        const uint32_t first = c * kSortChunk, len = n - first < kSortChunk ? n - first : kSortChunk;
        place += keys_before(keys + first, len, key, c < mine);      // equal tokens of earlier chunks come first
    }
    out_keys[place] = key;
    out_positions[place] = positions[i];
}

// ------------------------------------------------------------------------------------------ summing the runs ----
// The sorted list is cut into pieces of kPiece entries, so that a token that fills a tenth of a batch is summed by
// many workgroups.  A run that lies in one piece goes straight to its row; of one that crosses a border every piece
// leaves a partial sum (slot 0: the run the piece begins in the middle of; slot 1: the run it ends in the middle
// of), which join_runs_kernel adds up in the pieces' order.
constexpr int kPiece = 32;
constexpr int kSumBlock = 64;              // one wavefront, eight elements a lane

struct SumArgs {
    const uint32_t *keys, *positions;
    uint32_t n, vocab, dim;
    int64_t dy_stride, out_stride;
    float scale;
    int accumulate;
    float *partial;                        // [piece][2][dim]
    DropoutParams d;
    bool in_aligned, out_aligned;
    uint32_t col_tiles, sum_blocks;
};

template <typename O>
__device__ inline void write_row(O *out, const SumArgs &a, uint32_t row, uint32_t col, float (&acc)[8])
{
    const int count = a.dim - col < 8 ? (int)(a.dim - col) : 8;
    const bool whole = a.out_aligned && count == 8;
    O *p = out + (int64_t)row * a.out_stride + col;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = acc[e] * a.scale;
    if (a.accumulate) {
        float old[8];
        load8(p, whole, count, old);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = old[e] + v[e];
    }
    store8(p, whole, count, v);
}

// Workgroups below sum_blocks sum a piece's columns; the others write zeros to the rows that no token names (there
// are none of those when the gradient is added to what is there).
template <typename T, typename O>
__global__ void __launch_bounds__(kSumBlock)
sum_runs_kernel(const T *dy, O *out, SumArgs a)
{
    if (blockIdx.x >= a.sum_blocks) {
        // 64 rows a workgroup: a lane looks one of them up, then the wavefront fills the absent ones together
        const uint32_t row = (blockIdx.x - a.sum_blocks) * 64 + threadIdx.x;
        bool absent = row < a.vocab;
        if (absent) {
            const uint32_t at = keys_before(a.keys, a.n, row, false);
            absent = at >= a.n || a.keys[at] != row;
        }
        uint64_t todo = __ballot(absent);
        const float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        while (todo) {
            const uint32_t r = row - threadIdx.x + (uint32_t)__builtin_ctzll(todo);
            todo &= todo - 1;
            for (uint32_t col = threadIdx.x * 8; col < a.dim; col += kSumBlock * 8) {
                const int count = a.dim - col < 8 ? (int)(a.dim - col) : 8;
                store8(out + (int64_t)r * a.out_stride + col, a.out_aligned && count == 8, count, zero);
            }
        }
        return;
    }
    const uint32_t piece = blockIdx.x / a.col_tiles;
    const uint32_t col = (blockIdx.x - piece * a.col_tiles) * (kSumBlock * 8) + threadIdx.x * 8;
    const uint32_t lo = piece * kPiece, hi = a.n - lo < kPiece ? a.n : lo + kPiece;
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
    constexpr uint32_t kAhead = 4;         // rows in flight a lane
    for (uint32_t i = 0; i < entries; i += kAhead) {
        float v[kAhead][8];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const uint32_t at = i + k < entries ? i + k : entries - 1;
            load8(dy + (int64_t)(uint32_t)__builtin_amdgcn_readlane(my_pos, at) * a.dy_stride + col, whole, count, v[k]);
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
            const uint32_t next = last ? (lo + entries == hi ? key_after : 0xFFFFFFFFu) : __builtin_amdgcn_readlane(my_key, at + 1);
            const bool goes_on = next == key;
            if (goes_on && !last) continue;        // (the last entry of a piece leaves its unfinished run behind)
            if (from_before || goes_on) {
                store8(a.partial + ((int64_t)piece * 2 + (from_before ? 0 : 1)) * a.dim + col, count == 8 && a.dim % 4 == 0, count, acc);
            } else if (count > 0) {
                write_row(out, a, key, col, acc);
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
    const uint32_t border = (piece + 1) * kPiece;      // (the grid leaves the last piece out: border < n)
    const uint32_t key = a.keys[border - 1];
    if (key == 0xFFFFFFFFu || a.keys[border] != key) return;
    const uint32_t lo = piece * kPiece;
    if (lo > 0 && a.keys[lo - 1] == key) return;       // it began in an earlier piece
    if (col >= a.dim) return;
    const uint32_t end = border + keys_before(a.keys + border, a.n - border, key, true);
    const uint32_t last = (end - 1) / kPiece;
    const int count = a.dim - col < 8 ? (int)(a.dim - col) : 8;
    const bool whole = count == 8 && a.dim % 4 == 0;
    float acc[8];
    load8(a.partial + ((int64_t)piece * 2 + 1) * a.dim + col, whole, count, acc);
    for (uint32_t c = piece + 1; c <= last; c++) {
        float v[8];
        load8(a.partial + (int64_t)c * 2 * a.dim + col, whole, count, v);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] = acc[e] + v[e];
    }
    write_row(out, a, key, col, acc);
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
    s.partial = at, at += n > kPiece ? up((n + kPiece - 1) / kPiece * 2 * dim * 4) : 0;
    s.bytes = at;
    return s;
}

template <typename T, typename O>
static void launch_sums(const SumArgs &a, uintptr_t dy, uintptr_t out, uint32_t grid, uint32_t join_grid, hipStream_t stream)
{
    if (grid) sum_runs_kernel<T, O><<<grid, kSumBlock, 0, stream>>>(reinterpret_cast<const T *>(dy), reinterpret_cast<O *>(out), a);
    if (join_grid) join_runs_kernel<O><<<join_grid, kSumBlock, 0, stream>>>(reinterpret_cast<O *>(out), a);
}

template <typename T>
static void launch_lookup(uintptr_t table, uintptr_t tokens, uintptr_t out, int n, int vocab, int dim, int table_stride,
                          int out_stride, float scale, const DropoutParams &d, hipStream_t stream)
{
    const bool aligned = (table | out) % 16 == 0 && (size_t)table_stride * sizeof(T) % 16 == 0 && (size_t)out_stride * sizeof(T) % 16 == 0;
    const uint32_t per_row = ((uint32_t)dim + 7) / 8;
    const uint32_t grid = (uint32_t)(((uint64_t)n * per_row + kLookupBlock - 1) / kLookupBlock);
    lookup_kernel<T><<<grid, kLookupBlock, 0, stream>>>(reinterpret_cast<const T *>(table), reinterpret_cast<const int *>(tokens),
                                                        reinterpret_cast<T *>(out), (uint32_t)n, (uint32_t)vocab, (uint32_t)dim,
                                                        per_row, table_stride, out_stride, scale, d, aligned);
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
    if (((uint64_t)num_tokens * (((uint32_t)dim + 7) / 8) + kLookupBlock - 1) / kLookupBlock > 0x7FFFFFFFull) {
        set_error("a lookup of %d rows of %d elements needs more workgroups than one launch can address", num_tokens, dim);
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
    if (num_tokens < 0 || vocab_size <= 0 || dim <= 0) return 0;
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
    const uint64_t pieces = ((uint64_t)n + kPiece - 1) / kPiece;
    const uint64_t fill = accumulate ? 0 : ((uint64_t)vocab_size + 63) / 64;
    if (pieces * a.col_tiles + fill > 0x7FFFFFFFull || ((uint64_t)n + kSortChunk - 1) / kSortChunk > 65535) {
        set_error("a gradient of %d rows of %d elements needs more workgroups than one launch can address", num_tokens, dim);
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
    if (n > 0) {
        const bool chunks = n > kSortChunk;
        uint32_t *to_keys = chunks ? reinterpret_cast<uint32_t *>(workspace + space.chunk_keys) : keys;
        uint32_t *to_positions = chunks ? reinterpret_cast<uint32_t *>(workspace + space.chunk_positions) : positions;
        const uint32_t longest = chunks ? kSortChunk : n;
        const dim3 grid((longest + kSortRows - 1) / kSortRows, (n + kSortChunk - 1) / kSortChunk);
        sort_chunk_kernel<<<grid, kSortRows * kSortSlices, 0, stream>>>(reinterpret_cast<const int *>(token_buffer), n,
                                                                        (uint32_t)vocab_size, padding_token, to_keys, to_positions);
        if (chunks) merge_chunks_kernel<<<(n + 255) / 256, 256, 0, stream>>>(to_keys, to_positions, n, keys, positions);
    }
    a.keys = keys;
    a.positions = positions;
    a.n = n;
    a.vocab = (uint32_t)vocab_size;
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
    const uint32_t grid = a.sum_blocks + (uint32_t)fill, join_grid = pieces > 1 ? (uint32_t)(pieces - 1) * a.col_tiles : 0;
    const auto launch = data_type == kFloat32                                       ? launch_sums<float, float>
                        : data_type == kFloat16 && gradient_type == kFloat16        ? launch_sums<_Float16, _Float16>
                        : data_type == kFloat16                                     ? launch_sums<_Float16, float>
                        : gradient_type == kBFloat16                                ? launch_sums<__bf16, __bf16>
                                                                                    : launch_sums<__bf16, float>;
    launch(a, output_gradient_buffer, table_gradient_buffer, grid, join_grid, stream);
    return hip_ok(hipGetLastError(), "embedding gradient launch") ? 0 : kRcHip;
} catch (...) {
    note_exception();
    return kRcHip;
}

}  // extern "C"
