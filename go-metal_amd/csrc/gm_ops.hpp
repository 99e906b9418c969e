// What the operators at the two ends of a language model's training step share: element types, the checks
// of their arguments, and the generator behind dropout.
#pragma once

#include "gm_context.hpp"

#include <cstdint>

namespace gm {

// Type codes of memory/tensor.go:12-17, and one for bfloat16.
enum : int { kFloat32 = 0, kFloat16 = 2, kBFloat16 = 4 };

inline bool known_type(int t) { return t == kFloat32 || t == kFloat16 || t == kBFloat16; }
inline size_t type_bytes(int t) { return t == kFloat32 ? 4 : 2; }

// Return codes of these entry points.
enum : int {
    kRcDevice = -1, kRcQueue = -2, kRcNoGpu = -3, kRcNil = -4, kRcRange = -5, kRcHip = -6, kRcAmp = -16, kRcWorkspace = -18,
    kRcType = -19,
};

// The context's GPU for the length of a call; the caller's current device comes back afterwards.  An error that some
// earlier HIP call left on the thread is dropped: what hipGetLastError() says behind the launches is about them alone.
class DeviceScope {
  public:
    explicit DeviceScope(Context *ctx)
    {
        if (!hip_ok(hipGetDevice(&before_), "hipGetDevice")) return;
        ok_ = before_ == ctx->device_id || make_current(ctx);
        changed_ = ok_ && before_ != ctx->device_id;
        (void)hipGetLastError();
    }
    ~DeviceScope()
    {
        if (changed_) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    bool ok() const { return ok_; }

  private:
    int before_ = 0;
    bool ok_ = false, changed_ = false;
};

// Whether rows x cols elements, `stride` apart from row to row, lie inside the allocation (handles of this
// library that are the start of one; of any other address the length is not known).
inline bool rows_fit(const char *what, uintptr_t buffer, size_t rows, size_t cols, size_t stride, size_t element)
{
    const size_t len = registry_length(buffer);
    if (len == 0 || rows == 0 || cols == 0) return true;
    if (((rows - 1) * stride + cols) * element <= len) return true;
    set_error("%s: %zu rows of %zu elements, %zu apart, exceed the %zu-byte buffer", what, rows, cols, stride, len);
    return false;
}

inline bool element_aligned(const char *what, uintptr_t buffer, size_t element)
{
    if (buffer % element == 0) return true;
    set_error("%s is not aligned for its elements", what);
    return false;
}

// ------------------------------------------------------------------ device side ----
template <typename T>
__device__ inline T from_float(float x)
{
    return (T)x;      // to nearest even; beyond the type's range to +-inf
}

// Eight consecutive elements as fp32.  `count` of them exist; whole: all eight, and the address is aligned to 16 bytes.
template <typename T>
__device__ inline void load8(const T *p, bool whole, int count, float (&v)[8])
{
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
    if (whole) {
#pragma unroll
        for (int h = 0; h < (int)(8 * sizeof(T) / 16); h++) {
            const Vec x = reinterpret_cast<const Vec *>(p)[h];
#pragma unroll
            for (int c = 0; c < (int)(16 / sizeof(T)); c++) v[h * (int)(16 / sizeof(T)) + c] = (float)x[c];
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = c < count ? (float)p[c] : 0.0f;
}

template <typename T>
__device__ inline void store8(T *p, bool whole, int count, const float (&v)[8])
{
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
    if (whole) {
#pragma unroll
        for (int h = 0; h < (int)(8 * sizeof(T) / 16); h++) {
            Vec x;
#pragma unroll
            for (int c = 0; c < (int)(16 / sizeof(T)); c++) x[c] = from_float<T>(v[h * (int)(16 / sizeof(T)) + c]);
            reinterpret_cast<Vec *>(p)[h] = x;
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < 8; c++)
        if (c < count) p[c] = from_float<T>(v[c]);
}

// Dropout's random bits: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// 2011), a function of its counter alone, so a mask is made again wherever it is needed and never stored.
// Counter of a block of eight elements: (block, block >> 32, site, step); key: the two seed words.  The four
// words give sixteen bits to each element, low halves first.
struct DropoutState {
    uint32_t seed_low, seed_high, step, reserved;
};

struct DropoutParams {
    const DropoutState *state;      // nullptr: no dropout
    uint32_t border;                // an element is kept when its 16 bits reach this (65536 p, rounded)
    float scale;                    // 65536 / (65536 - border), 0 when nothing is kept
    uint32_t site;
};

__device__ inline void philox(uint64_t block, uint32_t site, const DropoutState &st, uint32_t (&c)[4])
{
    uint32_t k0 = st.seed_low, k1 = st.seed_high;
    c[0] = (uint32_t)block;
    c[1] = (uint32_t)(block >> 32);
    c[2] = site;
    c[3] = st.step;
#pragma unroll
    for (int round = 0; round < 10; round++) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k0;
        c[1] = (uint32_t)b;
        c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k1;
        c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// v[0..8) are the elements first .. first + 7 of the tensor; those dropped become 0 whatever they were.
__device__ inline void drop8(float (&v)[8], uint64_t first, const DropoutParams &d, const DropoutState &st)
{
    uint32_t c[4];
    philox(first >> 3, d.site, st, c);
    const uint32_t shift = (uint32_t)first & 7u;
    if (shift == 0) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t bits = e & 1 ? c[e >> 1] >> 16 : c[e >> 1] & 0xFFFFu;
            v[e] = bits >= d.border ? v[e] * d.scale : 0.0f;
        }
        return;
    }
    // rows that are no multiple of eight long: the eight elements lie in two blocks
    uint32_t n[4];
    philox((first >> 3) + 1, d.site, st, n);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t at = shift + e;             // 0 .. 14 over both blocks
        uint32_t word = 0;
#pragma unroll
        for (int w = 0; w < 8; w++) word = (at >> 1) == (uint32_t)w ? (w < 4 ? c[w & 3] : n[w & 3]) : word;
        const uint32_t bits = at & 1u ? word >> 16 : word & 0xFFFFu;
        v[e] = bits >= d.border ? v[e] * d.scale : 0.0f;
    }
}

// probability in [0, 1]; NaN is not.
inline bool dropout_params(float probability, uintptr_t state, int site, DropoutParams *out)
{
    if (!(probability >= 0.0f && probability <= 1.0f)) {
        set_error("dropout probability %g is not in [0, 1]", (double)probability);
        return false;
    }
    out->border = (uint32_t)((double)probability * 65536.0 + 0.5);
    out->scale = out->border < 65536u ? (float)(65536.0 / (65536.0 - (double)out->border)) : 0.0f;
    out->site = (uint32_t)site;
    out->state = probability > 0.0f ? reinterpret_cast<const DropoutState *>(state) : nullptr;
    return true;
}

}  // namespace gm
