// Dropout of rows for gfx950, the mask recomputed from a counter wherever it is needed:
//
//   y[r][c] = residual[r][c] + kept(r C + c) * up * x[r][c]
//
// The gradient with respect to x is the same pass over dy without a residual, with the same
// (seed, step), so nothing is kept between the two.  See DropRows (nf_rows.h) for the mask.
//
// A thread takes one unit of eight columns = one block of the generator.  Bound by memory:
// x, the residual and y each move once; the seven rounds (14 products of 32 x 32 -> 64 bits)
// and eight comparisons of a unit fit under its loads and stores.  (32768 x 768 bf16 with a
// residual, 151 MB: 23 .. 28 us, 5.4 .. 6.4 TB/s out of the last-level cache; a large copy 4.9.)

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nf_rows.h"

using namespace nfd;

namespace {

constexpr long kMaxBlocks = (1L << 24) - 1;

template <class T, bool kRes>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, const T* res, T* y, long R, long C,
                                                      long ldx, long ldr, long ldy, long units,
                                                      long first_block, DropRows d) {
    const unsigned long u = static_cast<unsigned long>(first_block + blockIdx.x) * 256 + threadIdx.x;
    if (u >= static_cast<unsigned long>(R * units)) return;
    unsigned long r = 0, k = u;
    if (R > 1) {  // (uniform; a 64-bit division costs several times a 32-bit one)
        r = (R * units) >> 32 ? u / units : static_cast<unsigned>(u) / static_cast<unsigned>(units);
        k = u - r * units;
    }
    const long c = static_cast<long>(k) * 8;
    const int n = C - c >= 8 ? 8 : static_cast<int>(C - c);
    float f[8];
    load_unit(x + r * ldx + c, n, f);
    float g[8];
    if (kRes) load_unit(res + r * ldr + c, n, g);
    if (d.limit != 0) drop8(d, drop_step(d), d.first + static_cast<long>(r) * C + c, f);
    if (kRes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += g[i];
    }
    store_unit(y + r * ldy + c, n, f);
}

template <class T>
int launch(const void* x, const void* res, void* y, long R, long C, long ldx, long ldr, long ldy,
           const DropRows& d, hipStream_t s) {
    const long units = (C + 7) / 8;
    const long blocks = (R * units + 255) / 256;
    // (a launch holds fewer than 2^32 threads)
    for (long b0 = 0; b0 < blocks; b0 += kMaxBlocks) {
        const dim3 grid(static_cast<unsigned>(blocks - b0 < kMaxBlocks ? blocks - b0 : kMaxBlocks));
        if (res != nullptr)
            hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(256), 0, s,
                               static_cast<const T*>(x), static_cast<const T*>(res),
                               static_cast<T*>(y), R, C, ldx, ldr, ldy, units, b0, d);
        else
            hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(256), 0, s,
                               static_cast<const T*>(x), nullptr, static_cast<T*>(y), R, C, ldx, 0L,
                               ldy, units, b0, d);
        const int status = static_cast<int>(hipGetLastError());
        if (status != 0) return status;
    }
    return 0;
}

}  // namespace

extern "C" {

// One argument block instead of fifteen arguments, whose conversion costs the caller more than the
// launch.  type: 0 float, 1 bf16, 2 half.  Rows of C columns, ld elements apart; y may be x or the
// residual (with the same distance between rows).  step_at: the step number in device memory,
// or null for `step`.  first: flattened index of the first element.
struct DropoutArgs {
    const void *x, *res;
    void* y;
    const long* step_at;
    long R, C, ldx, ldr, ldy, first;
    unsigned long long seed;
    unsigned limit, step;
    int type, unused;
};

int nf_dropout_args_size() { return static_cast<int>(sizeof(DropoutArgs)); }

int nf_dropout(const DropoutArgs* args, hipStream_t s) {
    const DropoutArgs& a = *args;
    if (a.R <= 0 || a.C <= 0 || a.limit > 65535u || a.first < 0) return -1;
    if (a.R > 1 && (a.ldx < a.C || a.ldy < a.C || (a.res != nullptr && a.ldr < a.C))) return -2;
    const DropRows d = {a.seed, a.step_at, a.step, a.limit, 65536.f / static_cast<float>(65536u - a.limit), a.first};
    switch (a.type) {
    case 0: return launch<float>(a.x, a.res, a.y, a.R, a.C, a.ldx, a.ldr, a.ldy, d, s);
    case 1: return launch<bf16>(a.x, a.res, a.y, a.R, a.C, a.ldx, a.ldr, a.ldy, d, s);
    case 2: return launch<half>(a.x, a.res, a.y, a.R, a.C, a.ldx, a.ldr, a.ldy, d, s);
    default: return -1;
    }
}

}  // extern "C"
