// Rows of 16-bit or 32-bit floats in units of eight columns, and the dropout mask of a unit.
#pragma once

#include "nf_device.h"
#include "../common/philox.h"

namespace nfd {

typedef _Float16 half;

// Eight elements at an address that is aligned to one element only: rows of odd length and
// column slices start anywhere, and the memory system takes 16-byte accesses at any address.
typedef bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef half halfx8u __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void load8(const bf16* p, float (&f)[8]) {
    const bf16x8u a = *reinterpret_cast<const bf16x8u*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(a[i]);
}
__device__ __forceinline__ void load8(const half* p, float (&f)[8]) {
    const halfx8u a = *reinterpret_cast<const halfx8u*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(a[i]);
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
    const f32x4u a = *reinterpret_cast<const f32x4u*>(p), b = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
}
__device__ __forceinline__ void store8(bf16* p, const float (&f)[8]) {
    bf16x8u a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = static_cast<bf16>(f[i]);
    *reinterpret_cast<bf16x8u*>(p) = a;
}
__device__ __forceinline__ void store8(half* p, const float (&f)[8]) {
    halfx8u a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = static_cast<half>(f[i]);
    *reinterpret_cast<halfx8u*>(p) = a;
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    f32x4u a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = f[i]; b[i] = f[4 + i]; }
    *reinterpret_cast<f32x4u*>(p) = a;
    *reinterpret_cast<f32x4u*>(p + 4) = b;
}

// The first n (1..8) of eight columns; the others read as 0 and are not written.
template <class T>
__device__ __forceinline__ void load_unit(const T* p, int n, float (&f)[8]) {
    if (n == 8) {
        load8(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? static_cast<float>(p[i]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store_unit(T* p, int n, const float (&f)[8]) {
    if (n == 8) {
        store8(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = static_cast<T>(f[i]);
    }
}

// Dropout of rows: element e of the flattened tensor is kept where the 16-bit half e & 7 of the
// block with counter (e >> 3 : 64 bits, 0, step) is at least `limit`; what is kept is scaled by
// `up` = 65536 / (65536 - limit).  limit 0: nothing is dropped.
struct DropRows {
    unsigned long seed;
    const long* step_at;  // the step number in device memory (a captured launch reads the
    unsigned step;        // present one at every replay), or null: `step`
    unsigned limit;
    float up;
    long first;           // flattened index of the tensor's first element
};

__device__ __forceinline__ unsigned drop_step(const DropRows& d) {
    return d.step_at != nullptr ? static_cast<unsigned>(*d.step_at) : d.step;
}

// f[i] = kept(e + i) ? f[i] * up : 0 for eight consecutive elements.  What is dropped is set to
// 0 whatever it was (also an infinity or a NaN).  A unit that starts inside a block of eight
// (rows of a length that is no multiple of 8) takes two blocks.
__device__ __forceinline__ void drop8(const DropRows& d, unsigned step, long e, float (&f)[8]) {
    const int sh = static_cast<int>(e & 7);
    const unsigned long b = static_cast<unsigned long>(e >> 3);
    const nf::Philox4 r = nf::philox4x32_7(d.seed, static_cast<unsigned>(b),
                                           static_cast<unsigned>(b >> 32), 0u, step);
    if (sh == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned h = (i & 1) ? r.v[i >> 1] >> 16 : r.v[i >> 1] & 0xFFFFu;
            f[i] = h >= d.limit ? f[i] * d.up : 0.f;
        }
        return;
    }
    const unsigned long b2 = b + 1;
    const nf::Philox4 q = nf::philox4x32_7(d.seed, static_cast<unsigned>(b2),
                                           static_cast<unsigned>(b2 >> 32), 0u, step);
    unsigned kept = 0;  // bit i: half i of the two blocks
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned h = (i & 1) ? r.v[i >> 1] >> 16 : r.v[i >> 1] & 0xFFFFu;
        const unsigned g = (i & 1) ? q.v[i >> 1] >> 16 : q.v[i >> 1] & 0xFFFFu;
        kept |= (h >= d.limit ? 1u << i : 0u) | (g >= d.limit ? 256u << i : 0u);
    }
    kept >>= sh;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (kept >> i) & 1u ? f[i] * d.up : 0.f;
}

}  // namespace nfd
