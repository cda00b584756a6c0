// Dropout whose mask is a function of (seed, position) and never stored.
//
// One Philox4x32-10 block decides eight elements, sixteen bits each (a rate is rounded down to a multiple of 2^-16 and
// what is kept is divided by the share that is really kept, so the expectation is exact): a thread takes the eight
// elements of one block, one 16-byte access of a 16-bit type or two of fp32.  Nothing but x and out moves: 65 536 000 elements
// of bf16 take 48 us, 5.5 TB/s, which is what a copy of 128 MiB reaches; 60 800 of fp32 take a launch (7 us with the call).
#include "ops_common.h"

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kDropoutTag = 0x50000000u;       // third counter word: no draw of the sampler or of the plan has it

template <class T> struct alignas(16) Eight { T x[8]; };

template <class T, bool ALIGNED>
__global__ __launch_bounds__(kThreads)
void dropout_kernel(const T *x, int64_t n, uint32_t threshold, float scale, uint64_t seed, const uint64_t *seed_device,
                    uint64_t offset, T *out) {
    if (seed_device) seed = seed_device[0];
    const int64_t n8 = (n + 7) / 8;
    for (int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x; b < n8; b += (int64_t)gridDim.x * kThreads) {
        const uint64_t c = offset + (uint64_t)b;
        uint32_t w[4];
        gs::philox4x32_10((uint32_t)c, (uint32_t)(c >> 32), kDropoutTag, 0u, (uint32_t)seed, (uint32_t)(seed >> 32), w);
        const bool whole = ALIGNED && b * 8 + 8 <= n;
        Eight<T> v;
        if (whole) v = reinterpret_cast<const Eight<T> *>(x)[b];
        else
            for (int i = 0; i < 8; ++i) v.x[i] = b * 8 + i < n ? x[b * 8 + i] : (T)0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t piece = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
            v.x[i] = piece >= threshold ? (T)((float)v.x[i] * scale) : (T)0.f;
        }
        if (whole) reinterpret_cast<Eight<T> *>(out)[b] = v;
        else
            for (int i = 0; i < 8; ++i)
                if (b * 8 + i < n) out[b * 8 + i] = v.x[i];
    }
}

template <class T>
int launch(const void *x, int64_t n, uint32_t threshold, float scale, uint64_t seed, const uint64_t *seed_device,
           uint64_t offset, void *out, hipStream_t stream) {
    int64_t blocks = ((n + 7) / 8 + kThreads - 1) / kThreads;
    if (blocks > 256 * 32) blocks = 256 * 32;
    const bool aligned = (((uintptr_t)x | (uintptr_t)out) & 15) == 0;
    hipLaunchKernelGGL((aligned ? dropout_kernel<T, true> : dropout_kernel<T, false>), dim3((unsigned)blocks), dim3(kThreads),
                       0, stream, static_cast<const T *>(x), n, threshold, scale, seed, seed_device, offset,
                       static_cast<T *>(out));
    return gs::check_launch("gs_dropout");
}

}  // namespace

extern "C" int gs_dropout(const void *x, int64_t n, int dtype, double rate, uint64_t seed, const uint64_t *seed_device,
                          uint64_t offset, void *out, void *stream) {
    const int size = gs::dtype_size(dtype);
    if (n < 0 || !size) return gs::fail(GS_EINVAL, "gs_dropout: n=%lld dtype=%d", (long long)n, dtype);
    if (!(rate >= 0.0) || !(rate * 65536.0 < 65536.0)) return gs::fail(GS_EINVAL, "gs_dropout: rate %g outside [0, 1)", rate);
    if (n == 0) return GS_OK;
    if (!x || !out) return gs::fail(GS_EINVAL, "gs_dropout: null pointer argument");
    if ((((uintptr_t)x | (uintptr_t)out) & (size - 1)) || ((uintptr_t)seed_device & 7))
        return gs::fail(GS_EINVAL, "gs_dropout: pointer not aligned to its element");
    if (n > INT64_MAX / 8) return gs::fail(GS_ELIMIT, "gs_dropout: n=%lld", (long long)n);
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)out, bytes = (uintptr_t)n * size;
    if (a != b && a < b + bytes && b < a + bytes) return gs::fail(GS_EINVAL, "gs_dropout: x and out overlap in part");
    const uint32_t threshold = (uint32_t)(rate * 65536.0);
    const float scale = (float)(65536.0 / (65536.0 - (double)threshold));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == GS_F32) return launch<float>(x, n, threshold, scale, seed, seed_device, offset, out, s);
    if (dtype == GS_BF16) return launch<__bf16>(x, n, threshold, scale, seed, seed_device, offset, out, s);
    return launch<_Float16>(x, n, threshold, scale, seed, seed_device, offset, out, s);
}
