// Dropout from a counter-based generator: y = keep ? x / (1 - p) : 0, plus a residual.  The mask is a function of
// (seed, step, site, element), so the backward pass is the same call on the gradient and nothing is stored.
#include "gm_ops.hpp"

#include "../../include/gometal_hip.h"

namespace gm {

constexpr int kDropBlock = 256;

// One lane makes one generator block: eight elements, 16 bytes of a 16-bit type a stream.  Memory bounds it, with
// the generator's ten rounds behind the loads: 33.6M fp16 with a residual, 201 MB, 35.6 us = 5.7 TB/s; 67M bf16 at an odd
// length, 269 MB, 44.4 us = 6.0 TB/s; 257000 fp32 2.8 us, a launch's latency.
template <typename T>
__global__ void __launch_bounds__(kDropBlock)
dropout_kernel(const T *x, const T *residual, T *y, uint32_t n, DropoutParams d, bool aligned)
{
    const uint64_t first = ((uint64_t)blockIdx.x * kDropBlock + threadIdx.x) * 8;
    if (first >= n) return;
    const int count = n - first < 8 ? (int)(n - first) : 8;
    const bool whole = aligned && count == 8;
    float v[8];
    load8(x + first, whole, count, v);
    if (d.state) {
        const DropoutState st = *d.state;
        drop8(v, first, d, st);
    }
    if (residual) {
        float r[8];
        load8(residual + first, whole, count, r);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = v[e] + r[e];
    }
    store8(y + first, whole, count, v);
}

__global__ void rng_advance_kernel(DropoutState *st) { st->step += 1; }

template <typename T>
static void launch_dropout(uintptr_t x, uintptr_t residual, uintptr_t y, int n, const DropoutParams &d, hipStream_t stream)
{
    const bool aligned = (x | residual | y) % 16 == 0;
    const unsigned int grid = ((unsigned int)n + kDropBlock * 8 - 1) / (kDropBlock * 8);
    dropout_kernel<T><<<grid, kDropBlock, 0, stream>>>(reinterpret_cast<const T *>(x), reinterpret_cast<const T *>(residual),
                                                       reinterpret_cast<T *>(y), (uint32_t)n, d, aligned);
}

}  // namespace gm

using namespace gm;

extern "C" {

int execute_dropout(uintptr_t device, uintptr_t command_queue, uintptr_t input_buffer, uintptr_t residual_buffer,
                    uintptr_t output_buffer, int num_elements, int data_type, float probability, uintptr_t rng_state, int site)
try {
    clear_error();
    if (device == 0) return kRcDevice;
    if (input_buffer == 0 || output_buffer == 0 || (rng_state == 0 && probability > 0.0f)) return kRcNil;
    if (!known_type(data_type)) return kRcType;
    DropoutParams d;
    if (num_elements < 0 || !dropout_params(probability, rng_state, site, &d)) return kRcRange;
    const size_t element = type_bytes(data_type), n = (size_t)num_elements;
    if (!element_aligned("input", input_buffer, element) || !element_aligned("residual", residual_buffer, element) ||
        !element_aligned("output", output_buffer, element) || !element_aligned("generator state", rng_state, 16) ||
        !rows_fit("input", input_buffer, 1, n, n, element) || !rows_fit("residual", residual_buffer, 1, n, n, element) ||
        !rows_fit("output", output_buffer, 1, n, n, element) || !rows_fit("generator state", rng_state, 1, 4, 4, 4))
        return kRcRange;
    Context *ctx = resolve_device(device);
    if (!ctx) return kRcNoGpu;
    hipStream_t stream;
    if (!queue_stream(ctx, command_queue, &stream)) return kRcQueue;
    if (n == 0) return 0;
    DeviceScope scope(ctx);
    if (!scope.ok()) return kRcHip;
    if (data_type == kFloat32) launch_dropout<float>(input_buffer, residual_buffer, output_buffer, num_elements, d, stream);
    else if (data_type == kFloat16) launch_dropout<_Float16>(input_buffer, residual_buffer, output_buffer, num_elements, d, stream);
    else launch_dropout<__bf16>(input_buffer, residual_buffer, output_buffer, num_elements, d, stream);
    return hip_ok(hipGetLastError(), "dropout launch") ? 0 : kRcHip;
} catch (...) {
    note_exception();
    return kRcHip;
}

int gm_rng_state_advance(uintptr_t device, uintptr_t command_queue, uintptr_t rng_state)
try {
    clear_error();
    if (device == 0) return kRcDevice;
    if (rng_state == 0) return kRcNil;
    if (!element_aligned("generator state", rng_state, 16) || !rows_fit("generator state", rng_state, 1, 4, 4, 4)) return kRcRange;
    Context *ctx = resolve_device(device);
    if (!ctx) return kRcNoGpu;
    hipStream_t stream;
    if (!queue_stream(ctx, command_queue, &stream)) return kRcQueue;
    DeviceScope scope(ctx);
    if (!scope.ok()) return kRcHip;
    rng_advance_kernel<<<1, 1, 0, stream>>>(reinterpret_cast<DropoutState *>(rng_state));
    return hip_ok(hipGetLastError(), "generator state launch") ? 0 : kRcHip;
} catch (...) {
    note_exception();
    return kRcHip;
}

}  // extern "C"
