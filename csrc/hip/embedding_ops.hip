// Embedding lookup with scaling, positions and dropout, and its gradient by sorted tokens,
// for gfx950.  float, bf16 and half tables; sums in fp32.
//
//   x[r]    = drop(scale * W[t_r] + P[r mod T])
//   dW[v]   = scale * sum over {r : t_r = v, v != padding} of drop'(dx[r])
//   dP[t]   = sum over b of drop'(dx[b T + t])
//
// A token outside [0, V) looks up a row of zeros and has no gradient.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nf_rows.h"

using namespace nfd;

namespace {

constexpr long kMaxBlocks = (1L << 24) - 1;

// A thread takes one unit of eight columns of one row.
template <class T>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const long* tokens, const T* table,
                                                            const T* pos, T* out, long R, long Tn,
                                                            long V, long C, long units, float scale,
                                                            long first_block, DropRows d) {
    const unsigned long u = static_cast<unsigned long>(first_block + blockIdx.x) * 256 + threadIdx.x;
    if (u >= static_cast<unsigned long>(R * units)) return;
    const bool wide = (R * units) >> 32;
    const long r = wide ? u / units : static_cast<unsigned>(u) / static_cast<unsigned>(units);
    const long c = (static_cast<long>(u) - r * units) * 8;
    const int n = C - c >= 8 ? 8 : static_cast<int>(C - c);
    const long tok = tokens[r];
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (tok >= 0 && tok < V) {
        load_unit(table + tok * C + c, n, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= scale;
    }
    if (pos != nullptr) {
        float g[8];
        const long t = wide ? r % Tn : static_cast<unsigned>(r) % static_cast<unsigned>(Tn);
        load_unit(pos + t * C + c, n, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += g[i];
    }
    if (d.limit != 0) drop8(d, drop_step(d), d.first + r * C + c, f);
    store_unit(out + r * C + c, n, f);
}

// Order by token: the place of row i is the number of rows with a smaller token, or the same
// token and a smaller index.
__global__ void __launch_bounds__(256) rank_kernel(const long* tokens, long V, long padding,
                                                   unsigned* key, unsigned* order, int R) {
    __shared__ unsigned ks[256];
    const int i = blockIdx.x * 256 + threadIdx.x;
    auto key_of = [&](int j) {
        const long t = tokens[j];
        return t < 0 || t >= V || t == padding ? static_cast<unsigned>(V) : static_cast<unsigned>(t);
    };
    const unsigned mine = i < R ? key_of(i) : 0u;
    int place = 0;
    for (int j0 = 0; j0 < R; j0 += 256) {
        __syncthreads();
        if (j0 + static_cast<int>(threadIdx.x) < R) ks[threadIdx.x] = key_of(j0 + threadIdx.x);
        __syncthreads();
        const int m = R - j0 < 256 ? R - j0 : 256;
        for (int j = 0; j < m; ++j) place += ks[j] < mine || (ks[j] == mine && j0 + j < i);
    }
    if (i < R) {
        key[place] = mine;
        order[place] = static_cast<unsigned>(i);
    }
}

template <class T>
__global__ void __launch_bounds__(256) zero_kernel(T* p, long n) {
    for (long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x; i < n;
         i += static_cast<long>(gridDim.x) * 256)
        p[i] = static_cast<T>(0.f);
}

// One wave per sorted position and 512 columns; the first position of a run sums it.
template <class T, class G>
__global__ void __launch_bounds__(256) embedding_bwd_kernel(const unsigned* key, const unsigned* order,
                                                            const T* dx, G* dw, int R, long V, long C,
                                                            int slabs, float scale, int accumulate,
                                                            DropRows d) {
    const int lane = threadIdx.x & 63;
    const long w = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int i = static_cast<int>(w / slabs);
    if (i >= R) return;
    const unsigned k = key[i];
    if (k >= static_cast<unsigned>(V) || (i > 0 && key[i - 1] == k)) return;
    const long c = (w % slabs) * 512 + lane * 8;
    if (c >= C) return;
    const int n = C - c >= 8 ? 8 : static_cast<int>(C - c);
    const unsigned step = drop_step(d);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = i; j < R && key[j] == k; ++j) {
        const long r = order[j];
        if (r >= R) continue;  // (no row: an order that is not of these tokens)
        float f[8];
        load_unit(dx + r * C + c, n, f);
        if (d.limit != 0) drop8(d, step, d.first + r * C + c, f);
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += f[q];
    }
    float old[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (accumulate) load_unit(dw + k * C + c, n, old);
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = fmaf(acc[q], scale, old[q]);
    store_unit(dw + k * C + c, n, acc);
}

template <class T, class G>
__global__ void __launch_bounds__(256) positions_bwd_kernel(const T* dx, G* dp, long B, long Tn, long C,
                                                            int slabs, DropRows d) {
    const int lane = threadIdx.x & 63;
    const long w = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const long t = w / slabs;
    const long c = (w % slabs) * 512 + lane * 8;
    if (t >= Tn || c >= C) return;
    const int n = C - c >= 8 ? 8 : static_cast<int>(C - c);
    const unsigned step = drop_step(d);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (long b = 0; b < B; ++b) {
        const long e = (b * Tn + t) * C + c;
        float f[8];
        load_unit(dx + e, n, f);
        if (d.limit != 0) drop8(d, step, d.first + e, f);
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += f[q];
    }
    store_unit(dp + t * C + c, n, acc);
}

inline DropRows drop_rows(unsigned limit, unsigned long long seed, const long* step_at, unsigned step,
                          long first) {
    return {seed, step_at, step, limit, 65536.f / static_cast<float>(65536u - limit), first};
}

template <class T>
int fwd(const long* tokens, const void* table, const void* pos, void* out, long R, long Tn, long V,
        long C, float scale, const DropRows& d, hipStream_t s) {
    const long units = (C + 7) / 8, blocks = (R * units + 255) / 256;
    for (long b0 = 0; b0 < blocks; b0 += kMaxBlocks) {
        const dim3 grid(static_cast<unsigned>(blocks - b0 < kMaxBlocks ? blocks - b0 : kMaxBlocks));
        hipLaunchKernelGGL((embedding_fwd_kernel<T>), grid, dim3(256), 0, s, tokens,
                           static_cast<const T*>(table), static_cast<const T*>(pos),
                           static_cast<T*>(out), R, Tn, V, C, units, scale, b0, d);
        const int status = static_cast<int>(hipGetLastError());
        if (status != 0) return status;
    }
    return 0;
}

template <class T, class G>
int bwd(const unsigned* key, const unsigned* order, const void* dx, void* dw, void* dp, long B, long Tn,
        long V, long C, float scale, int accumulate, const DropRows& d, hipStream_t s) {
    const int slabs = static_cast<int>((C + 511) / 512);
    const long R = B * Tn;
    if (!accumulate)
        hipLaunchKernelGGL((zero_kernel<G>), dim3(4096), dim3(256), 0, s, static_cast<G*>(dw), V * C);
    hipLaunchKernelGGL((embedding_bwd_kernel<T, G>), dim3(static_cast<unsigned>((R * slabs + 3) / 4)),
                       dim3(256), 0, s, key, order, static_cast<const T*>(dx), static_cast<G*>(dw),
                       static_cast<int>(R), V, C, slabs, scale, accumulate, d);
    if (dp != nullptr)
        hipLaunchKernelGGL((positions_bwd_kernel<T, G>), dim3(static_cast<unsigned>((Tn * slabs + 3) / 4)),
                           dim3(256), 0, s, static_cast<const T*>(dx), static_cast<G*>(dp), B, Tn, C,
                           slabs, d);
    return static_cast<int>(hipGetLastError());
}

}  // namespace

extern "C" {

// tokens: R ids; table [V][C]; pos (may be null): [>= T][C], row r takes position r mod T.
// type: 0 float, 1 bf16, 2 half (table, pos and out).
int nf_embedding_fwd(const long* tokens, const void* table, const void* pos, void* out, int type,
                     long R, long T, long V, long C, float scale, unsigned limit,
                     unsigned long long seed, const long* step_at, unsigned step, long first,
                     hipStream_t s) {
    if (R <= 0 || T <= 0 || V <= 0 || C <= 0 || limit > 65535u || first < 0) return -1;
    const DropRows d = drop_rows(limit, seed, step_at, step, first);
    switch (type) {
    case 0: return fwd<float>(tokens, table, pos, out, R, T, V, C, scale, d, s);
    case 1: return fwd<bf16>(tokens, table, pos, out, R, T, V, C, scale, d, s);
    case 2: return fwd<half>(tokens, table, pos, out, R, T, V, C, scale, d, s);
    default: return -1;
    }
}

// key[i]: the i-th smallest token (V: none, or the padding token), order[i]: its row; equal
// tokens in the order of their rows.
int nf_token_order(const long* tokens, unsigned* key, unsigned* order, long R, long V, long padding,
                   hipStream_t s) {
    if (R <= 0 || R >= (1L << 31) || V <= 0 || V >= (1L << 31)) return -1;
    hipLaunchKernelGGL(rank_kernel, dim3(static_cast<unsigned>((R + 255) / 256)), dim3(256), 0, s,
                       tokens, V, padding, key, order, static_cast<int>(R));
    return static_cast<int>(hipGetLastError());
}

// key / order: from nf_token_order.  dx: B T rows of C.  dw [V][C]: written everywhere, or
// (accumulate) added to where tokens are.  dp (may be null): rows 0 .. T - 1 are written.
// type: of dx; grad_type: of dw and dp (0, or the type of dx).
int nf_embedding_bwd(const unsigned* key, const unsigned* order, const void* dx, void* dw, void* dp,
                     int type, int grad_type, long B, long T, long V, long C, float scale,
                     int accumulate, unsigned limit, unsigned long long seed, const long* step_at,
                     unsigned step, long first, hipStream_t s) {
    if (B <= 0 || T <= 0 || V <= 0 || C <= 0 || limit > 65535u || first < 0) return -1;
    if (B * T >= (1L << 31) || B * T * ((C + 511) / 512) >= (1L << 32)) return -3;
    if (grad_type != 0 && grad_type != type) return -1;
    const DropRows d = drop_rows(limit, seed, step_at, step, first);
    switch (type * 4 + grad_type) {
    case 0: return bwd<float, float>(key, order, dx, dw, dp, B, T, V, C, scale, accumulate, d, s);
    case 4: return bwd<bf16, float>(key, order, dx, dw, dp, B, T, V, C, scale, accumulate, d, s);
    case 5: return bwd<bf16, bf16>(key, order, dx, dw, dp, B, T, V, C, scale, accumulate, d, s);
    case 8: return bwd<half, float>(key, order, dx, dw, dp, B, T, V, C, scale, accumulate, d, s);
    case 10: return bwd<half, half>(key, order, dx, dw, dp, B, T, V, C, scale, accumulate, d, s);
    default: return -1;
    }
}

}  // extern "C"
