// gdn2_dropout_*: y = x / (1 - p) or 0, by the words of philox.hpp.
//
// Rows that lie together, of a multiple of 8 channels, are one row (their counters
// follow one another); a thread takes a run of 16 bytes.  Other rows go in runs of VEC
// channels from each row's start, the last one shorter; loads and stores need no
// alignment.
//
// Bound: HBM, the generator beside it.  32768 x 2048 bfloat16: 42 us alone, 45 in turn
// with other work, 6.0 TB/s (four runs a thread, all loaded first: 48); 2331 x 1537 f32,
// whose rows start anywhere: 6.3 us, 4.6 TB/s.
#include <algorithm>
#include <exception>
#include <string>

#include "common.hpp"
#include "gdn2_block.h"
#include "loose_io.hpp"
#include "philox.hpp"

namespace gdn2 {
namespace {

template <typename T, int VEC> __global__ __launch_bounds__(256) void dropout_flat_kernel(const T *x, T *y, int64_t n, Drop d) {
    drop_begin(d);
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
    if (i >= n) return;
    const Raw<T, VEC> r = loose<T, VEC>(x + i);
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)r[j];
    drop_n<VEC>(d, (uint64_t)i / 4, d.scale, v);
    loose_store<T, VEC>(y + i, v);
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void dropout_rows_kernel(const T *x, T *y, uint32_t runs, uint32_t runs_a_row, int64_t C,
                                                           int64_t sx, int64_t sy, Drop d) {
    drop_begin(d);
    const uint64_t quads = (uint64_t)(C + 3) / 4, run = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (run >= runs) return;
    const uint32_t row = (uint32_t)run / runs_a_row, c = ((uint32_t)run - row * runs_a_row) * VEC;
    float v[VEC];
    load_part<T, VEC>(x + row * sx + c, C - c, v);
    drop_n<VEC>(d, row * quads + c / 4, d.scale, v);
    store_part<T, VEC>(y + row * sy + c, C - c, v);
}

template <typename T> gdn2_status run(const void *x, void *y, int64_t rows, int64_t C, int64_t sx, int64_t sy,
                                      const gdn2_dropout *drop, hipStream_t s, const char *name) {
    constexpr int VEC = 16 / sizeof(T);
    const std::string who = std::string(name) + ": ";
    if (rows < 0 || C < 0) return fail(GDN2_EINVAL, who + "negative dimension");
    if (!drop || !drop_ok(*drop)) return fail(GDN2_EINVAL, who + "p must be between 0 and 1");
    if (rows == 0 || C == 0) return GDN2_OK;
    if (!x || !y) return fail(GDN2_EINVAL, who + "null pointer");
    if (x == y && rows > 1 && sx != sy) return fail(GDN2_EINVAL, who + "in place, the strides must be equal");
    const Drop d = drop_of(*drop);
    const double quads = (double)rows * (double)((C + 3) / 4);
    if (C >= (int64_t(1) << 31) || rows >= (int64_t(1) << 40))
        return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
    if (C % 8 == 0 && (rows == 1 || (sx == C && sy == C))) {
        const int64_t per = 256 * VEC;
        // (fewer than 2^24 workgroups, 2^32 threads; in doubles: the product may pass 64 bits)
        if ((double)rows * (double)C > ((1 << 24) - 1) * (double)per)
            return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
        const int64_t n = rows * C, blocks = (n + per - 1) / per;
        hipLaunchKernelGGL((dropout_flat_kernel<T, VEC>), dim3((unsigned)blocks), dim3(256), 0, s, static_cast<const T *>(x),
                           static_cast<T *>(y), n, d);
    } else {
        if (quads >= 4294967040.) return fail(GDN2_NOT_APPLICABLE, who + "sizes above the kernels' limits");
        const int64_t runs_a_row = (C + VEC - 1) / VEC, runs = rows * runs_a_row;
        hipLaunchKernelGGL((dropout_rows_kernel<T, VEC>), dim3((unsigned)((runs + 255) / 256)), dim3(256), 0, s,
                           static_cast<const T *>(x), static_cast<T *>(y), (uint32_t)runs, (uint32_t)runs_a_row, C, sx, sy, d);
    }
    GDN2_HIP_CHECK(hipGetLastError());
    return GDN2_OK;
}

}  // namespace
}  // namespace gdn2

#define GDN2_ENTRY(suffix, T)                                                                                            \
    extern "C" gdn2_status gdn2_dropout_##suffix(const void *x, void *y, int64_t rows, int64_t channels, int64_t stride_x, \
                                                 int64_t stride_y, const gdn2_dropout *drop, gdn2_stream_t stream) {     \
        try { /* no exception leaves a C entry */                                                                        \
            return gdn2::run<T>(x, y, rows, channels, stride_x, stride_y, drop, (hipStream_t)stream,                     \
                                "gdn2_dropout_" #suffix);                                                                \
        } catch (const std::exception &) {                                                                               \
            return GDN2_EHIP;                                                                                            \
        }                                                                                                                \
    }
GDN2_ENTRY(f32, float)
GDN2_ENTRY(bf16, gdn2::bf16)
