// Attention of any length and layout for gfx950, forward and backward, with dropped
// probabilities: bf16 or half, head dimensions 8 .. 128 (multiples of 8), strided q / k / v,
// heads that share keys and values, a length per sequence.
//
//   S = scale * Q K^T over the keys a query sees: key j of query i where j < n and (causal)
//       j <= i + n - m   (m queries and n keys of the sequence: the last query sees every key)
//   P = softmax(S),  O = (kept * up * P) V,  lse = log sum exp S
//
//   D  = rowsum(dO * O)                       dV = (kept * up * P)^T dO
//   dS = P * (kept * up * (dO V^T) - D)       dQ = scale * dS K      dK = scale * dS^T Q
//
// The probabilities (and the dropout mask) are computed again in the backward pass from lse and
// from the counter; neither is ever stored.  Rows i >= m and rows that see no key give 0 (lse
// -inf), their gradients are 0 too, and what q, k, v, dout hold beyond m and n is not used, so it
// may be anything.  dK and dV of shared heads are summed in registers over the heads in turn.
//
// The score tiles are 32 keys x 32 queries, S^T = K Q^T in the forward and dQ kernels (a query
// per lane: its softmax statistics stay in the lane) and S = Q K^T in the dK / dV kernel (a key
// per lane), so that every probability tile leaves the accumulator straight as an operand of the
// next MFMA; the other operand comes through transposing LDS reads in the accumulator's order.
// A tile sits in LDS once: its 16-byte pieces are permuted so that neither the row reads nor the
// transposing reads meet bank conflicts (nfix::attn_off).
//
// The mask: probability (i, j) of head h of sequence b takes byte j & 3 of word i & 3 of the block
// with counter (j >> 2, i >> 2, b * heads + h, step) and is kept where it is at least `limit`
// (p = limit / 256).  A 4 x 4 block serves both layouts: the four lanes of a quad need the same
// four blocks of a 32-row tile, each computes one and they exchange words, so a 32 x 32 tile
// costs every lane one block for its 16 probabilities.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "../common/philox.h"
#include "nf_device.h"

using namespace nfd;

namespace {

typedef _Float16 half;
typedef half halfx8 __attribute__((ext_vector_type(8)));
typedef half halfx4 __attribute__((ext_vector_type(4)));

template <class E> struct Vec;
template <> struct Vec<bf16> { typedef bf16x8 x8; typedef bf16x4 x4; };
template <> struct Vec<half> { typedef halfx8 x8; typedef halfx4 x4; };

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(halfx8 a, halfx8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x4 tr4(const bf16* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16(NF_LDS(bf16x4, p));
}
__device__ __forceinline__ halfx4 tr4(const half* p) {
    typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
    const fp16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4f16(NF_LDS(fp16x4, p));
    return __builtin_bit_cast(halfx4, v);
}

constexpr int kStage = 64;  // keys (or queries) per LDS stage
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Half has the exponents 2^-14 .. 2^15 (2^-24 with fewer bits), and the factors P and dS = P (dP - D) of the
// gradients leave them long before the gradients do: P is 1 / keys, dS that times dO.  So the backward
// kernels hold P times 2^kProb, which a probability cannot carry beyond the type, and dS times a power of
// two on top, which the dQ kernel finds for every query from what it meets (GradScale), the dK / dV kernel for
// its workgroup from what the dQ kernel left (bounds).  Both are exact and are taken out in fp32.  bf16
// has the exponents of fp32 and needs neither.
//
// In the forward pass the reference that scores are taken relative to follows the running maximum only
// where that gets ahead by a factor of 2^kSlack in the probability: any reference gives the same quotients,
// and what the sums so far would have to be multiplied by at nearly every tile (some of 32 rows finds a new
// maximum) is spared.  bf16 has room for any slack.  In half what a probability is below the largest one
// costs bits from 2^-14 on, and 2^22 keys of 2^-26 have 1 / 16 of the largest one's weight: there P carries
// 2^kLift (so do the sums, which cancel it), and the slack is what is left of the type: 2^(3 + 12).
template <class E> struct Exponent {
    static constexpr bool kScaled = false;
    static constexpr float kProb = 0.f, kUnprob = 1.f;  // 2^-kProb
    static constexpr float kSlack = 8.f, kLift = 0.f;
};
template <> struct Exponent<half> {
    static constexpr bool kScaled = true;
    static constexpr float kProb = 15.f, kUnprob = 1.f / 32768.f;
    static constexpr float kSlack = 3.f, kLift = 12.f;
};

struct Strides { long b, t, h; };  // elements between sequences, rows, heads

struct AttnArgs {
    const void* q; Strides sq;
    const void* k; Strides sk;
    const void* v; Strides sv;
    void* out; Strides so;
    const void* dout; Strides sdo;
    void* dq; Strides sdq;
    void* dk; Strides sdk;
    void* dv; Strides sdv;
    float* lse;               // [B][H][Tq]
    float* delta;             // [B][H][Tq], rowsum(dO * O): written by the dQ kernel; bounds behind it
    const int *qlen, *klen;   // [B] or null
    const long* step_at;
    unsigned long seed;
    unsigned long first_head; // number of the first head of the mask's counter
    int B, Tq, Tk, H, Hk, D, causal;
    float scale, up;
    unsigned limit, step;
    float* parts;             // partial results of key chunks (few queries) or query ranges (dK / dV)
    int target;               // few queries: workgroups to cut the keys for (0: not cut)
    int splits;               // dK / dV: query ranges at most
};

// -- tiles ------------------------------------------------------------------------------------
// R rows of DP columns in LDS.  They come through registers by buffer loads: the descriptor starts
// at the tile's first row and ends with the last row there is, so rows behind it (and, by an offset
// beyond any tile, columns behind D) read as 0 without a comparison, and a lane keeps one 32-bit
// offset per piece for the whole loop.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <class E, int DP, int R>
struct Tile {
    typedef typename Vec<E>::x8 x8;
    typedef typename Vec<E>::x4 x4;
    static constexpr int kRow = DP * 2, kBytes = R * kRow;
    static constexpr int kPieces = DP / 8;             // 16-byte pieces of a row
    static constexpr int kPer = R * kPieces / 256;     // ... per thread (256 threads)
    struct Regs { u32x4 v[kPer]; };
    struct From {                                      // a matrix that is walked tile by tile
        const E* base;
        long ld;
        int rows, D;
        unsigned off[kPer];
    };

    static __device__ __forceinline__ From from(const void* p, long first, long ld, int rows, int D, int tid) {
        From f = {static_cast<const E*>(p) + first, ld, rows, D, {}};
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int idx = tid + 256 * i, c = (idx % kPieces) * 8;
            f.off[i] = c < D ? static_cast<unsigned>((idx / kPieces) * ld + c) * 2u : 0x80000000u;
        }
        return f;
    }
    static __device__ __forceinline__ Regs load(const From& f, int tile) {
        const int left = f.rows - tile * R;
        const long bytes = left > 0 ? ((min(left, R) - 1) * f.ld + f.D) * 2 : 0;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<E*>(f.base + tile * R * f.ld), 0, static_cast<int>(bytes), 0x00020000);
        Regs t;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            t.v[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, static_cast<int>(f.off[i]), 0, 0);
        return t;
    }
    static __device__ __forceinline__ void store(char* lds, const Regs& t, int tid) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int idx = tid + 256 * i;
            *reinterpret_cast<u32x4*>(lds + nfix::attn_off(DP, idx / kPieces, idx % kPieces)) = t.v[i];
        }
    }

    // Operand fragments.  The permutation of the pieces has a period of 16 rows, so a lane's
    // offsets within 16 (or 32) rows are computed once and the rest is a constant.
    struct Lane {
        int row[DP / 16];     // row (lane & 31), columns 16 ks + 8 (lane >> 5) .. + 7
        int tr[DP / 32][2];   // transposing reads of columns 32 i + (lane & 31)
    };
    static __device__ __forceinline__ Lane lane_offsets(int lane) {
        Lane o;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) o.row[ks] = nfix::attn_off(DP, lane & 31, 2 * ks + (lane >> 5));
        const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2), x = 16 * ((lane >> 4) & 1) + 4 * (i & 3);
#pragma unroll
        for (int j = 0; j < DP / 32; ++j) {
            o.tr[j][0] = nfix::attn_off(DP, r, (32 * j + x) >> 3) + (x & 7) * 2;
            o.tr[j][1] = nfix::attn_off(DP, r + 8, (32 * j + x) >> 3) + (x & 7) * 2;
        }
        return o;
    }
    // rows row0 + (lane & 31); row0 a multiple of 32
    static __device__ __forceinline__ x8 row(const char* lds, const Lane& o, int row0, int ks) {
        return *reinterpret_cast<const x8*>(lds + row0 * kRow + o.row[ks]);
    }
    // 8 values tile[k0 + (j & 3) + 4 h + 8 (j >> 2)][32 i + (lane & 31)], h = lane >> 5, k0 a multiple
    // of 16: rows in the order in which an accumulator hands them to the next MFMA
    static __device__ __forceinline__ x8 tr(const char* lds, const Lane& o, int k0, int i) {
        const x4 lo = tr4(reinterpret_cast<const E*>(lds + k0 * kRow + o.tr[i][0]));
        const x4 hi = tr4(reinterpret_cast<const E*>(lds + k0 * kRow + o.tr[i][1]));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// rows [.., D) of a lane's own row as operand fragments, 0 where there is no row or column
template <class E, int DP>
__device__ __forceinline__ void own_row(const E* p, bool there, int D, int hh, typename Vec<E>::x8 (&f)[DP / 16]) {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        f[ks] = {};
        const int c = ks * 16 + 8 * hh;
        if (there && c < D) f[ks] = *reinterpret_cast<const typename Vec<E>::x8*>(p + c);
    }
}

template <class E>
__device__ __forceinline__ typename Vec<E>::x8 pack8(const f32x16& v, int first) {
    typename Vec<E>::x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = static_cast<E>(v[first + j]);
    return o;
}

// what pack8 rounds away
template <class E>
__device__ __forceinline__ typename Vec<E>::x8 rest8(const f32x16& v, int first) {
    typename Vec<E>::x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = static_cast<E>(v[first + j] - static_cast<float>(static_cast<E>(v[first + j])));
    return o;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// -- the dropout mask of a 32 x 32 tile -------------------------------------------------------
template <int kCtrl>
__device__ __forceinline__ unsigned quad(unsigned v) {
    return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xF, 0xF, true));
}

// w[j] of lane t <- w[t] of lane j, within each four lanes
__device__ __forceinline__ void quad_transpose(unsigned (&w)[4], int lane) {
    const bool o1 = lane & 1, o2 = lane & 2;
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const unsigned x = quad<0xB1>(o1 ? w[k] : w[k + 1]);  // lane ^ 1
        if (o1) w[k] = x; else w[k + 1] = x;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const unsigned x = quad<0x4E>(o2 ? w[k] : w[k + 2]);  // lane ^ 2
        if (o2) w[k] = x; else w[k + 2] = x;
    }
}

// The factor of a query's dS: so that the largest one of the first tile with any lies in [2^6, 2^7), and
// room for those that are up to 2^8 times larger; where a tile holds one beyond that, what was summed so far
// is multiplied too.  (A narrower room costs: with a factor of 4 to 8 some of a wave's 32 rows pass it every
// few tiles, and the dQ kernel of six sequences of up to 777, 16 heads on 4 of 128, takes 58 us instead of
// 55.  Without any of this it takes 49.5, the dK / dV kernel 61 instead of 63.)
struct GradScale {
    float x = 1.f, limit = 0.f, top = 0.f;  // |dS * x| up to `top` so far, `limit` allowed (0: all dS so far are 0)

    // The further factor for a tile whose largest |dS * x| of this query is `most`.
    __device__ __forceinline__ float grow(float most) {
        if (!(most > limit)) return 1.f;  // (also a NaN)
        if (most == INFINITY) {           // the row's gradient is not finite, whatever the factor
            limit = INFINITY;
            return 1.f;
        }
        // (at most 2^60: with it no dO V^T of half operands passes the range of fp32)
        const float f = ldexpf(1.f, min(7 - __builtin_amdgcn_frexp_expf(most), 60));
        x *= f;
        top *= f;
        limit = 32768.f;
        return f;
    }
    __device__ __forceinline__ bool set() const { return limit == 32768.f; }
};

// Bytes of the lane's 16 probabilities, four per word: byte e of word g belongs to accumulator
// register 4 g + e.  kKeysInRows: the rows of the tile are keys (row0 = first key, col0 = first
// query), else queries.
template <bool kKeysInRows>
__device__ __forceinline__ void mask_bytes(unsigned (&w)[4], unsigned long seed, unsigned head,
                                           unsigned step, int row0, int col0, int lane) {
    const unsigned rows = (row0 >> 2) + 2 * (lane & 3) + (lane >> 5), cols = (col0 >> 2) + ((lane & 31) >> 2);
    const nf::Philox4 r = kKeysInRows ? nf::philox4x32_7(seed, rows, cols, head, step)
                                      : nf::philox4x32_7(seed, cols, rows, head, step);
    if (kKeysInRows) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = r.v[j];   // word = query & 3 = lane & 3 of the taker
    } else {
        // word = query & 3 = the register, byte = key & 3 = the taker: transpose the 4 x 4 bytes
        const unsigned a = __builtin_amdgcn_perm(r.v[1], r.v[0], 0x05010400u);  // 1.1 0.1 1.0 0.0
        const unsigned b = __builtin_amdgcn_perm(r.v[1], r.v[0], 0x07030602u);
        const unsigned c = __builtin_amdgcn_perm(r.v[3], r.v[2], 0x05010400u);
        const unsigned d = __builtin_amdgcn_perm(r.v[3], r.v[2], 0x07030602u);
        w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
        w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
        w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
        w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
    }
    quad_transpose(w, lane);
}

__device__ __forceinline__ bool kept(const unsigned (&w)[4], int r, unsigned limit) {
    return ((w[r >> 2] >> (8 * (r & 3))) & 0xFFu) >= limit;
}

// Tiles that every query of the wave sees whole are most of them; without this the comparisons
// of the others would be turned into selects that all tiles pay for.
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// Keeps a group of LDS reads together and ahead of what follows.  Left alone the compiler puts every
// read right before the MFMA that takes it, into the same registers, and each product then waits
// for an LDS round trip.
__device__ __forceinline__ void reads_first() { __builtin_amdgcn_sched_barrier(0); }

// row of accumulator register r without the lane's part (4 (lane >> 5))
__device__ __forceinline__ constexpr int reg_row(int r) { return (r & 3) + 8 * (r >> 2); }

// of a lane and its other half (lane ^ 32)
__device__ __forceinline__ float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// of all lanes
__device__ __forceinline__ float max_wave(float v) {
    auto with = [&](unsigned other) { v = fmaxf(v, __uint_as_float(other)); };
    with(quad<0xB1>(__float_as_uint(v)));   // lane ^ 1
    with(quad<0x4E>(__float_as_uint(v)));   // lane ^ 2
    with(quad<0x141>(__float_as_uint(v)));  // the other four of eight, mirrored
    with(quad<0x140>(__float_as_uint(v)));  // the other eight of sixteen, mirrored
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    return max_halves(v);
}
__device__ __forceinline__ float sum_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// -- what a workgroup knows about its sequence -------------------------------------------------
struct Seq { int m, n, off; };  // queries, keys, and: query i sees keys j <= i + off

__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
    Seq s;
    s.m = a.qlen != nullptr ? min(max(a.qlen[b], 0), a.Tq) : a.Tq;
    s.n = a.klen != nullptr ? min(max(a.klen[b], 0), a.Tk) : a.Tk;
    s.off = a.causal ? s.n - s.m : 0x3FFFFFFF;
    return s;
}
__device__ __forceinline__ int keys_seen(const Seq& s, int i) {  // (i + off fits: i < 2^30)
    return min(s.n, max(0, i + s.off + 1));
}

// What a tile of 128 keys reads in the dK / dV kernel: per head the stages from the first one with a
// query that sees a key of it (query i sees key j from i >= j - off on), and the ranges that these
// stages of all heads are cut into.
// Stages that a range of the dK / dV kernel has at least (6 ragged sequences of up to 777, 16 heads on
// 4: 56.7 us with 6 and 62 with 10 at 64 columns, where two workgroups share a CU; 105 and 98 at 128).
__host__ __device__ constexpr int least_range(int D) { return D > 64 ? 10 : 6; }

struct KeyPlan { int first, per, ranges; };

__device__ __forceinline__ KeyPlan key_plan(const AttnArgs& a, const Seq& s, int tile0) {
    if (tile0 >= s.n) return {0, 0, 1};
    const int first = a.causal ? max(0, tile0 - s.off) / kStage : 0;
    const int per = max(0, (s.m + kStage - 1) / kStage - first);
    return {first, per, min(a.splits, max(1, (per * (a.H / a.Hk) + least_range(a.D) - 1) / least_range(a.D)))};
}

// The sequence and head of a workgroup, `heads` of them per sequence.  Workgroups go to the XCDs and to
// the quarters of each in turn, whatever these have to do: where lengths differ the sequences are
// shifted by one from tile to tile, or every tile of a sequence would go to the same place.  (The dQ
// kernel on six lengths of 0 .. 777: 51 .. 63 us by their order, 47 .. 53 shifted.)
__device__ __forceinline__ int shifted_head(const AttnArgs& a, int heads) {
    if (a.klen == nullptr && a.qlen == nullptr) return blockIdx.x;
    return static_cast<int>((blockIdx.x + static_cast<unsigned long>(heads) * blockIdx.y) % gridDim.x);
}

__host__ __device__ __forceinline__ long delta_floats(const AttnArgs& a) {
    return (static_cast<long>(a.B) * a.H * a.Tq + 3) & ~3L;
}
// Behind delta: for every 32 queries of a head a bound of 2^kProb |dS| (half).
__host__ __device__ __forceinline__ int bounds_of_head(const AttnArgs& a) { return (a.Tq + 31) / 32; }
__host__ __device__ __forceinline__ long bound_floats(const AttnArgs& a) {
    return (static_cast<long>(a.B) * a.H * bounds_of_head(a) + 3) & ~3L;
}

__device__ __forceinline__ unsigned step_of(const AttnArgs& a) {
    return a.step_at != nullptr ? static_cast<unsigned>(*a.step_at) : a.step;
}

// ---------------------------------------------------------------------------------------------
// Forward: one workgroup = 128 queries (4 waves x 32) of one head; tiles of 64 keys, double-
// buffered in LDS.  grid = (sequence and head, tile): the tiles of a head land on one XCD, the
// long ones are dispatched first.  Two sequences of 4096, 12 heads of 64: 82 us = 620 TFLOP/s of the
// pairs seen; 32 x 1024 x 12 with dropout: 122 us.  P is rounded to the operands' type for the product (the
// matrix unit takes no other), once, relative to a reference near the row's maximum; maximum, sum and O stay
// in fp32: the output is 1.2 .. 1.4 times as far off as rounding it leaves.  Bound by the vector work on
// the probabilities (an exponential, a maximum, a sum and a rounding each, half as much again with the mask) beside the
// two products, at the 1.9 GHz that the chip holds under it.
//
// KG = 2: a workgroup has 64 queries and two waves for each 32 of them, which take the even and the
// odd tiles of keys and are joined through LDS at the end.  Twice as many workgroups of half the
// length, for launches that the longest workgroup would hold up (see halve_keys).
template <class E, int DP, bool kDrop, int KG>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu((DP == 64 ? 4 : 3) - KG)))
attn_fwd_kernel(AttnArgs a) {
    typedef Tile<E, DP, kStage> T;
    typedef typename T::x8 x8;
    typedef Exponent<E> X;
    constexpr int NB = DP / 32, W = 4 / KG, kQueries = 32 * W;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int bh = shifted_head(a, a.H), b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hk);
    const int tile0 = (gridDim.y - 1 - blockIdx.y) * kQueries;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hh = lane >> 5;
    const Seq sq = sequence(a, b);
    const int grp = __builtin_amdgcn_readfirstlane(wave / W), q0 = tile0 + wave % W * 32, qi = q0 + n;
    const int stages = tile0 < sq.m ? (keys_seen(sq, min(tile0 + kQueries - 1, sq.m - 1)) + kStage - 1) / kStage : 0;
    const typename T::From kfrom = T::from(a.k, b * a.sk.b + hk * a.sk.h, a.sk.t, sq.n, a.D, tid);
    const typename T::From vfrom = T::from(a.v, b * a.sv.b + hk * a.sv.h, a.sv.t, sq.n, a.D, tid);
    const typename T::Lane at = T::lane_offsets(lane);
    x8 qf[DP / 16];
    own_row<E, DP>(static_cast<const E*>(a.q) + b * a.sq.b + h * a.sq.h + qi * a.sq.t, qi < sq.m, a.D, hh, qf);
    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x16{0};
    float m = -INFINITY, l = 0.f, msc = 0.f;  // running maximum, sum, and maximum in the exponent
    const float sc2 = a.scale * kLog2e;
    // keys that the wave's first and last query see, and this lane's (less its rows' offset)
    const int seen_lo = __builtin_amdgcn_readfirstlane(keys_seen(sq, q0)), seen = keys_seen(sq, qi) - 4 * hh;
    const int seen_hi = __builtin_amdgcn_readfirstlane(q0 < sq.m ? keys_seen(sq, q0 + 31) : 0);
    const unsigned step = kDrop ? step_of(a) : 0u, head = static_cast<unsigned>(a.first_head + bh);

    typename T::Regs kr[KG], vr[KG];
    constexpr int kBuf = 2 * KG * T::kBytes;
    auto tile = [&](const char* Ks, const char* Vs, int key0) {
        f32x16 s[2] = {{0}, {0}};
#pragma unroll
        for (int part = 0; part < DP / 64; ++part) {
            x8 f[2][4];
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) f[sub][ks] = T::row(Ks, at, sub * 32, 4 * part + ks);
            reads_first();
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) s[sub] = mma(f[sub][ks], qf[4 * part + ks], s[sub]);
        }
        if (key0 + kStage > seen_lo) {  // wave-uniform: some pair of the tile is not visible
            keep_branch();
            const int lim = seen - key0;
#pragma unroll
            for (int r = 0; r < 32; ++r)
                if (reg_row(r & 15) + 32 * (r >> 4) >= lim) s[r >> 4][r & 15] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int r = 1; r < 32; ++r) mx = fmaxf(mx, s[r >> 4][r & 15]);
        mx = max_halves(mx);
        if (__any((mx - m) * sc2 > X::kSlack)) {
            const float mn = fmaxf(m, mx);
            const float ref = mn == -INFINITY ? 0.f : mn;
            const float alpha = exp2_fast((m - ref) * sc2);
            m = mn;
            msc = ref * sc2 - X::kLift;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            x8 vf[2][NB];
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < NB; ++i) vf[g][i] = T::tr(Vs, at, sub * 32 + 16 * g, i);
            reads_first();
            float r0 = 0.f, r1 = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                s[sub][r] = exp2_fast(fmaf(s[sub][r], sc2, -msc));
                s[sub][r + 1] = exp2_fast(fmaf(s[sub][r + 1], sc2, -msc));
                r0 += s[sub][r];
                r1 += s[sub][r + 1];
            }
            l += r0 + r1;
            if (kDrop) {  // the sum is of all probabilities, what is dropped leaves the product
                unsigned w[4];
                mask_bytes<true>(w, a.seed, head, step, key0 + 32 * sub, q0, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!kept(w, r, a.limit)) s[sub][r] = 0.f;
            }
            const x8 p0 = pack8<E>(s[sub], 0), p1 = pack8<E>(s[sub], 8);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                o[i] = mma(vf[0][i], p0, o[i]);
                o[i] = mma(vf[1][i], p1, o[i]);
            }
        }
    };
    auto fetch = [&](int it) {
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            kr[g] = T::load(kfrom, it * KG + g);
            vr[g] = T::load(vfrom, it * KG + g);
        }
    };
    auto put = [&](char* to) {
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            T::store(to + 2 * g * T::kBytes, kr[g], tid);
            T::store(to + (2 * g + 1) * T::kBytes, vr[g], tid);
        }
    };
    const int turns = (stages + KG - 1) / KG;
    auto turn = [&](int it, char* here, char* there) {
        if (it + 1 < turns) fetch(it + 1);
        const int key0 = (it * KG + grp) * kStage;
        const char* at0 = here + 2 * grp * T::kBytes;
        if (key0 < seen_hi) tile(at0, at0 + T::kBytes, key0);  // wave-uniform
        if (it + 1 < turns) put(there);
        __syncthreads();
    };
    if (turns > 0) {
        fetch(0);
        put(smem);
    }
    __syncthreads();
    for (int it = 0; it < turns; it += 2) {
        turn(it, smem, smem + kBuf);
        if (it + 1 < turns) turn(it + 1, smem + kBuf, smem);
    }
    if (KG == 2) {
        float* park = reinterpret_cast<float*>(smem) + (wave % W) * 64 * (NB * 16 + 2) + lane;
        if (grp == 1) {
            park[0] = m;
            park[64] = l;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) park[64 * (2 + 16 * i + r)] = o[i][r];
        }
        __syncthreads();
        if (grp == 1) return;
        const float m2 = park[0], mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
        const float a1 = exp2_fast((m - ref) * sc2), a2 = exp2_fast((m2 - ref) * sc2);
        m = mn;
        l = l * a1 + park[64] * a2;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = o[i][r] * a1 + park[64 * (2 + 16 * i + r)] * a2;
    }
    if (qi >= a.Tq) return;
    l = sum_halves(l);
    const bool some = qi < sq.m && (l > 0.f || l != l);
    const float inv = some ? (kDrop ? a.up : 1.f) / l : 0.f;
    E* orow = static_cast<E*>(a.out) + b * a.so.b + qi * a.so.t + h * a.so.h;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            typename T::x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<E>(some ? o[i][4 * g + e] * inv : 0.f);
            const int c = 32 * i + 8 * g + 4 * hh;
            if (c < a.D) *reinterpret_cast<typename T::x4*>(orow + c) = v;
        }
    if (hh == 0)
        a.lse[static_cast<long>(bh) * a.Tq + qi] = some ? m * a.scale + kLn2 * (__builtin_amdgcn_logf(l) - X::kLift) : -INFINITY;
}

// ---------------------------------------------------------------------------------------------
// Forward of few queries against many keys: the queries of all heads that share a key head are the
// columns of one tile of 32, so the keys are read once for all of them (more than 32: once for each
// tile, blockIdx.y).  Bound by reading the keys and values.  A workgroup takes a chunk of the keys, its
// waves every fourth 32 of them, through LDS of their own (no barrier in the loop), one tile ahead
// in registers.  The waves are joined through LDS, the chunks by attn_join_kernel.
//
// The chunks are cut on the device, from the lengths: about `target` of equal size over all
// sequences, so a batch of short and long ones still fills the chip evenly.  What a chunk costs
// apart from its keys (the first load, the joins) is worth some hundred keys, so there are no more
// of them than workgroups run at once.  (Four caches of up to 8191 keys x 8 heads x 128, 84 MB:
// 18 .. 19 us + 5.1 us for the join with 512 workgroups, 4.4 .. 4.7 TB/s; 23.0 + 4.9 with 256; without the
// hint that the keys are read once, which leaves the parts in L2, 20.2 + 6.2.)
typedef float f32x2 __attribute__((ext_vector_type(2)));
constexpr int kFewQueries = 32, kFewRows = 256, kFewTarget = 512;
constexpr int kOnce = 2;  // non-temporal load

struct Chunk { int b, hk, count, at, size; Seq seq; };  // chunk `at` of `count` of (b, hk), keys per chunk

__device__ __forceinline__ int few_keys(const Seq& s) { return s.m > 0 ? s.n : 0; }

__device__ __forceinline__ int lane_sum(int v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Keys per chunk, given the number of keys of all sequences (B * Hk < target, so the sum of what
// the sequences' last chunks are short of adds less than `target` workgroups).
__device__ __forceinline__ int few_size(const AttnArgs& a, long keys) {
    return static_cast<int>(max(128L, ((keys * a.Hk + a.target - 1) / a.target + 127) & ~127L));
}

// Which chunk workgroup `id` has; b < 0: none.  All lanes; lane i looks at sequences i, i + 64, ...
__device__ __forceinline__ Chunk few_chunk(const AttnArgs& a, int id, int lane) {
    if (a.target == 0) return {id / a.Hk, id % a.Hk, 1, 0, a.Tk, sequence(a, id / a.Hk)};
    const Seq mine0 = lane < a.B ? sequence(a, lane) : Seq{0, 0, 0};
    long keys = few_keys(mine0);
    for (int i = lane + 64; i < a.B; i += 64) keys += few_keys(sequence(a, i));
    const int size = few_size(a, lane_sum(static_cast<int>(keys)));  // (fewer than 512 sequences of up to 2^22)
    int before = 0;  // parts of the sequences before
    for (int i0 = 0; i0 < a.B; i0 += 64) {
        const Seq mine = i0 == 0 ? mine0 : (i0 + lane < a.B ? sequence(a, i0 + lane) : Seq{0, 0, 0});
        const int count = (few_keys(mine) + size - 1) / size;
        int x = count;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int y = __shfl_up(x, off, 64);
            if (lane >= off) x += y;
        }
        const unsigned long here = __ballot(id < (before + x) * a.Hk);
        if (here != 0) {
            const int who = __builtin_ctzl(here), c = __builtin_amdgcn_readlane(count, who);
            const int at = id - (before + __builtin_amdgcn_readlane(x, who) - c) * a.Hk, k = at / a.Hk;
            const Seq s = {__builtin_amdgcn_readlane(mine.m, who), __builtin_amdgcn_readlane(mine.n, who),
                           __builtin_amdgcn_readlane(mine.off, who)};
            return {i0 + who, at - k * a.Hk, c, k, size, s};
        }
        before += __builtin_amdgcn_readlane(x, 63);
    }
    return {-1, 0, 0, 0, 0, {0, 0, 0}};
}

//
// kTwice: up to 16 rows (queries times heads that share a key head), so the tile's other 16 columns are
// free, and they undo the rounding of P: they hold the same rows again, as P less what the first ones round
// it to, and the joint adds them.  It costs the subtraction only, no product and no read.  (Error of one head
// of 64 against 680 keys over that of rounding the output: 1.0, without it 1.3 .. 1.5.)
template <class E, int DP, bool kTwice>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
attn_few_kernel(AttnArgs a) {
    typedef Tile<E, DP, 32> T;
    typedef typename T::x8 x8;
    typedef Exponent<E> X;
    constexpr int NB = DP / 32, KS = DP / 16, kPer = 32 * T::kPieces / 64;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, n = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Chunk me = few_chunk(a, blockIdx.x, lane);
    if (me.b < 0) return;
    const int b = me.b, hk = me.hk, group = a.H / a.Hk;
    const Seq sq = me.seq;
    const int row0 = 32 * blockIdx.y, all = a.Tq * group, rows = min(32, all - row0);  // of this tile
    const int own = kTwice ? n & 15 : n;  // row of the tile that this column has
    const int qi = (row0 + own) / group, h = hk * group + (row0 + own) % group;
    const bool in = own < rows && qi < sq.m;
    const float second = n < 16 ? 0.f : 1.f;
    const int seen = (in ? keys_seen(sq, qi) : 0) - 4 * hh;
    const int k0 = me.at * me.size, k1 = min(sq.m > 0 ? sq.n : 0, k0 + me.size);
    char* lds = smem + wave * 2 * T::kBytes;  // K, V
    const typename T::Lane at = T::lane_offsets(lane);
    x8 qf[KS];
    own_row<E, DP>(static_cast<const E*>(a.q) + b * a.sq.b + qi * a.sq.t + h * a.sq.h, in, a.D, hh, qf);
    unsigned koff[kPer], voff[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int idx = lane + 64 * i, r = idx / T::kPieces, c = (idx % T::kPieces) * 8;
        koff[i] = c < a.D ? static_cast<unsigned>(r * a.sk.t + c) * 2u : 0x80000000u;
        voff[i] = c < a.D ? static_cast<unsigned>(r * a.sv.t + c) * 2u : 0x80000000u;
    }
    const E* kb = static_cast<const E*>(a.k) + b * a.sk.b + hk * a.sk.h;
    const E* vb = static_cast<const E*>(a.v) + b * a.sv.b + hk * a.sv.h;
    u32x4 kr[kPer], vr[kPer];
    auto fetch = [&](int key0) {  // rows behind the last key read as 0
        const long last = min(sq.n - key0, 32) - 1;
        const __amdgpu_buffer_rsrc_t kd = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<E*>(kb + key0 * a.sk.t), 0, static_cast<int>((last * a.sk.t + a.D) * 2), 0x00020000);
        const __amdgpu_buffer_rsrc_t vd = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<E*>(vb + key0 * a.sv.t), 0, static_cast<int>((last * a.sv.t + a.D) * 2), 0x00020000);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            kr[i] = __builtin_amdgcn_raw_buffer_load_b128(kd, static_cast<int>(koff[i]), 0, kOnce);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            vr[i] = __builtin_amdgcn_raw_buffer_load_b128(vd, static_cast<int>(voff[i]), 0, kOnce);
    };
    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x16{0};
    float m = -INFINITY, l = 0.f, msc = 0.f;
    const float sc2 = a.scale * kLog2e;
    int key0 = k0 + wave * 32;
    if (key0 < k1) fetch(key0);
    for (; key0 < k1; key0 += 128) {
        // (the LDS operations of a wave complete in order: the reads of the tile before come first)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int idx = lane + 64 * i, to = nfix::attn_off(DP, idx / T::kPieces, idx % T::kPieces);
            *reinterpret_cast<u32x4*>(lds + to) = kr[i];
            *reinterpret_cast<u32x4*>(lds + T::kBytes + to) = vr[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (key0 + 128 < k1) fetch(key0 + 128);
        f32x16 s = {0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = mma(T::row(lds, at, 0, ks), qf[ks], s);
        const int lim = min(seen, k1 - 4 * hh) - key0;
        float mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (reg_row(r) >= lim) s[r] = -INFINITY;
            mx = fmaxf(mx, s[r]);
        }
        mx = max_halves(mx);
        if (__any((mx - m) * sc2 > X::kSlack)) {
            const float mn = fmaxf(m, mx);
            const float ref = mn == -INFINITY ? 0.f : mn;
            const float alpha = exp2_fast((m - ref) * sc2);
            m = mn;
            msc = ref * sc2 - X::kLift;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
        }
        float rs = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(fmaf(s[r], sc2, -msc));
            rs += s[r];
        }
        l += rs;
        if (kTwice) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fmaf(static_cast<float>(static_cast<E>(s[r])), -second, s[r]);
        }
        const x8 p0 = pack8<E>(s, 0), p1 = pack8<E>(s, 8);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            o[i] = mma(T::tr(lds + T::kBytes, at, 0, i), p0, o[i]);
            o[i] = mma(T::tr(lds + T::kBytes, at, 16, i), p1, o[i]);
        }
    }
    l = sum_halves(l);
    // Join the waves: each leaves its m, l and O [rows][DP] (where its tiles were; the 16-byte pieces
    // of a row permuted, as a row is a whole number of bank rounds), then all threads sum them.
    constexpr int kPieces = DP / 4;
    float* ml = reinterpret_cast<float*>(smem + 8 * T::kBytes);  // [wave][m, l][32]
    if (hh == 0) {
        ml[wave * 64 + n] = m;
        ml[wave * 64 + 32 + n] = l;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (own < rows) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = o[i][4 * g + e];
                *reinterpret_cast<f32x4*>(lds + (n * kPieces + ((8 * i + 2 * g + hh) ^ (n & (kPieces - 1)))) * 16) = v;
            }
    }
    __syncthreads();
    const long parts = static_cast<long>(gridDim.x) * all;
    for (int idx = threadIdx.x; idx < rows * kPieces; idx += 256) {
        const int row = idx / kPieces, piece = idx % kPieces, col = 4 * piece;
        float mw[4], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, mw[w] = ml[w * 64 + row]);
        const float ref = top == -INFINITY ? 0.f : top;
        f32x4 v = {0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = exp2_fast((mw[w] - ref) * sc2);
            sum = fmaf(ml[w * 64 + 32 + row], f, sum);
#pragma unroll
            for (int again = 0; again < (kTwice ? 32 : 16); again += 16) {
                const int at = row + again;
                const f32x4 part = *reinterpret_cast<const f32x4*>(
                    smem + w * 2 * T::kBytes + (at * kPieces + (piece ^ (at & (kPieces - 1)))) * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = fmaf(part[e], f, v[e]);
            }
        }
        if (me.count > 1) {
            const long part = static_cast<long>(blockIdx.x) * all + row0 + row;
            *reinterpret_cast<f32x4*>(a.parts + part * DP + col) = v;
            if (piece == 0) *reinterpret_cast<f32x2*>(a.parts + parts * DP + 2 * part) = f32x2{top, sum};
            continue;
        }
        const int qr = (row0 + row) / group, head = hk * group + (row0 + row) % group;
        const bool some = qr < sq.m && (sum > 0.f || sum != sum);
        const float inv = some ? 1.f / sum : 0.f;
        if (col < a.D) {
            typename T::x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = static_cast<E>(some ? v[e] * inv : 0.f);
            *reinterpret_cast<typename T::x4*>(static_cast<E*>(a.out) + b * a.so.b + qr * a.so.t + head * a.so.h + col) = y;
        }
        if (piece == 0)
            a.lse[(static_cast<long>(b) * a.H + head) * a.Tq + qr] =
                some ? top * a.scale + kLn2 * (__builtin_amdgcn_logf(sum) - X::kLift) : -INFINITY;
    }
}

// One wave per row of a sequence that was cut: the chunks' maxima and sums, 64 at a time, then
// their O in order.
template <class E, int DP>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, int workgroups) {
    const int lane = threadIdx.x & 63, group = a.H / a.Hk, rows = a.Tq * group;
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= a.B * a.Hk * rows) return;
    const int bh = row / rows, r = row % rows, b = bh / a.Hk, hk = bh % a.Hk;
    const int qi = r / group, h = hk * group + r % group;
    const Seq sq = sequence(a, b);
    int keys = 0, first = 0;  // keys of all sequences; parts of those before b
    for (int i = lane; i < a.B; i += 64) keys += few_keys(sequence(a, i));
    const int size = few_size(a, lane_sum(keys)), count = (few_keys(sq) + size - 1) / size;
    if (count == 1) return;  // written already
    for (int i = lane; i < b; i += 64) first += (few_keys(sequence(a, i)) + size - 1) / size;
    first = lane_sum(first) * a.Hk + hk;  // the parts of chunk c: first + c Hk
    const int live = qi < sq.m ? count : 0;
    const long parts = static_cast<long>(workgroups) * rows;
    const float sc2 = a.scale * kLog2e;
    const f32x2* ml = reinterpret_cast<const f32x2*>(a.parts + parts * DP);
    constexpr int kFlight = 8;  // parts in flight
    float v0[kFlight], v1[kFlight];
    auto pair = [&](int c) {
        return c < live ? ml[static_cast<long>(first + c * a.Hk) * rows + r] : f32x2{-INFINITY, 0.f};
    };
    auto load = [&](int c) {
        const float* o = a.parts + (static_cast<long>(first) * rows + r) * DP + lane;
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const float* oc = o + static_cast<long>(min(c + u, live - 1)) * a.Hk * rows * DP;
            v0[u] = oc[0];
            if (DP > 64) v1[u] = oc[64];
        }
    };
    f32x2 mine = pair(lane);
    if (live > 0) load(0);  // beside the maxima
    float m = mine[0];
    for (int c = lane + 64; c < live; c += 64) m = fmaxf(m, pair(c)[0]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int c0 = 0; c0 < live; c0 += 64) {
        if (c0 > 0) mine = pair(c0 + lane);
        const float w = exp2_fast((mine[0] - ref) * sc2);
        l = fmaf(mine[1], w, l);
        const int more = min(64, live - c0);
        for (int c1 = 0; c1 < more; c1 += kFlight) {
            if (c0 + c1 > 0) load(c0 + c1);
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                const float wc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), c1 + u));
                if (c1 + u < more) {
                    o0 = fmaf(v0[u], wc, o0);
                    if (DP > 64) o1 = fmaf(v1[u], wc, o1);
                }
            }
        }
    }
    l = wave_sum(l);
    const bool some = l > 0.f || l != l;
    const float inv = some ? 1.f / l : 0.f;
    E* orow = static_cast<E*>(a.out) + b * a.so.b + qi * a.so.t + h * a.so.h;
    if (lane < a.D) orow[lane] = static_cast<E>(some ? o0 * inv : 0.f);
    if (DP > 64 && 64 + lane < a.D) orow[64 + lane] = static_cast<E>(some ? o1 * inv : 0.f);
    if (lane == 0)
        a.lse[(static_cast<long>(b) * a.H + h) * a.Tq + qi] =
            some ? m * a.scale + kLn2 * (__builtin_amdgcn_logf(l) - Exponent<E>::kLift) : -INFINITY;
}

// ---------------------------------------------------------------------------------------------
// Backward, queries: four waves x 32 queries (KG = 2: two waves for each 32 of 64, as in the forward
// kernel); streams K / V.
//
// D = rowsum(dO * O) takes O as it was stored: rounded, and summed from rounded probabilities.
// Its error is the same for all keys of a row, so it would come back as error * (P K) in dQ and
// make dQ and dK half as far off again as the two roundings that they cannot do without.  But
// sum_j dS_ij = 0 in exact arithmetic, so the row's sum r = sum_j dS_ij, which costs one addition
// per pair in fp32, is that error: dQ is corrected by -r (P K), at the cost of a fourth product,
// and the dK / dV kernel that follows gets D + r.
//
// Both backward kernels on 32 x 1024 x 12 heads of 64 with dropout: 335 us (half: 351), bound like
// the forward one; at 128 columns the accumulators leave one wave per SIMD (8 x 1024 x 16 heads:
// 244 us), and a workgroup's time is 9 us + 1.2 us per 32 keys, which is what bounds ragged batches.
//
// kFine: P and dS are rounded to the operands' type for the products, an error like that of rounding
// the results, so that the two add up to sqrt(2) of one.  Short sequences undo it by a product with what
// the rounding left (see fine).
template <class E, int DP, bool kDrop, int KG, bool kFine>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP == 64 ? 2 : 1)))
attn_dq_kernel(AttnArgs a) {
    constexpr int R = kStage, NB = DP / 32, W = 4 / KG, kQueries = 32 * W;
    typedef Exponent<E> X;
    typedef Tile<E, DP, R> T;
    typedef typename T::x8 x8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int bh = shifted_head(a, a.H), b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hk);
    const int tile0 = (gridDim.y - 1 - blockIdx.y) * kQueries;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hh = lane >> 5;
    const Seq sq = sequence(a, b);
    const int grp = __builtin_amdgcn_readfirstlane(wave / W), q0 = tile0 + wave % W * 32, qi = q0 + n;
    const bool in = qi < sq.m;
    const int stages = tile0 < sq.m ? (keys_seen(sq, min(tile0 + kQueries - 1, sq.m - 1)) + R - 1) / R : 0;
    const typename T::From kfrom = T::from(a.k, b * a.sk.b + hk * a.sk.h, a.sk.t, sq.n, a.D, tid);
    const typename T::From vfrom = T::from(a.v, b * a.sv.b + hk * a.sv.h, a.sv.t, sq.n, a.D, tid);
    const typename T::Lane at = T::lane_offsets(lane);
    x8 qf[DP / 16], df[DP / 16];
    own_row<E, DP>(static_cast<const E*>(a.q) + b * a.sq.b + h * a.sq.h + qi * a.sq.t, in, a.D, hh, qf);
    own_row<E, DP>(static_cast<const E*>(a.dout) + b * a.sdo.b + h * a.sdo.h + qi * a.sdo.t, in, a.D, hh, df);
    float delta = 0.f;
    {
        x8 of[DP / 16];
        own_row<E, DP>(static_cast<const E*>(a.out) + b * a.so.b + h * a.so.h + qi * a.so.t, in, a.D, hh, of);
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                delta = fmaf(static_cast<float>(df[ks][j]), static_cast<float>(of[ks][j]), delta);
    }
    delta = sum_halves(delta);
    const long row = static_cast<long>(bh) * a.Tq + qi;
    // a row that sees no key has lse -inf: +inf makes its probabilities 0
    float lse2 = in ? a.lse[row] : -INFINITY;
    lse2 = lse2 == -INFINITY ? INFINITY : lse2 * kLog2e - X::kProb;
    GradScale gs;
    float up = kDrop ? a.up : 1.f, xdelta = delta;  // times gs.x
    f32x16 dq[NB], pk[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) { dq[i] = f32x16{0}; pk[i] = f32x16{0}; }
    float off = 0.f;  // sum of dS
    const float sc2 = a.scale * kLog2e;
    const int seen_lo = __builtin_amdgcn_readfirstlane(keys_seen(sq, q0)), seen = keys_seen(sq, qi) - 4 * hh;
    const int seen_hi = __builtin_amdgcn_readfirstlane(q0 < sq.m ? keys_seen(sq, q0 + 31) : 0);
    const unsigned step = kDrop ? step_of(a) : 0u, head = static_cast<unsigned>(a.first_head + bh);

    typename T::Regs kr[KG], vr[KG];
    constexpr int kBuf = 2 * KG * T::kBytes;
    auto tile = [&](const char* Ks, const char* Vs, int key0) {
        f32x16 s = {0}, dp = {0};
#pragma unroll
        for (int part = 0; part < DP / 64; ++part) {
            x8 f[4], e[4];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                f[ks] = T::row(Ks, at, 0, 4 * part + ks);
                e[ks] = T::row(Vs, at, 0, 4 * part + ks);
            }
            reads_first();
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                s = mma(f[ks], qf[4 * part + ks], s);
                dp = mma(e[ks], df[4 * part + ks], dp);
            }
        }
        x8 kt[2][NB];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int i = 0; i < NB; ++i) kt[g][i] = T::tr(Ks, at, 16 * g, i);
        reads_first();
        unsigned w[4];
        if (kDrop) mask_bytes<true>(w, a.seed, head, step, key0, q0, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(fmaf(s[r], sc2, -lse2));
            if (kDrop) dp[r] = fmaf(dp[r], kept(w, r, a.limit) ? up : 0.f, -xdelta);
            else if (X::kScaled) dp[r] = fmaf(dp[r], up, -xdelta);
            else dp[r] -= delta;
        }
        if (key0 + 32 > seen_lo) {  // wave-uniform: some pair of the tile is not visible
            keep_branch();
            const int lim = seen - key0;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (reg_row(r) >= lim) { s[r] = 0.f; dp[r] = 0.f; }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] *= s[r];
        if (X::kScaled) {
            float some[4] = {0.f, 0.f, 0.f, 0.f};  // (four short chains)
#pragma unroll
            for (int r = 0; r < 16; ++r) some[r & 3] = fmaxf(some[r & 3], fabsf(dp[r]));
            float most = fmaxf(fmaxf(some[0], some[1]), fmaxf(some[2], some[3]));
            if (__any(most > gs.limit)) {
                keep_branch();
                most = max_halves(most);  // (both halves of a query take the same factor)
                const float f = gs.grow(most);
                most *= f;
                up *= f;
                xdelta *= f;
                off *= f;
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= f;
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) dq[i][r] *= f;
            }
            gs.top = fmaxf(gs.top, most);
        }
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) t += dp[r];
        off += t;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const x8 ds = pack8<E>(dp, 8 * g), p = pack8<E>(s, 8 * g);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                dq[i] = mma(kt[g][i], ds, dq[i]);
                pk[i] = mma(kt[g][i], p, pk[i]);
            }
        }
        if (kFine) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const x8 ds = rest8<E>(dp, 8 * g);
#pragma unroll
                for (int i = 0; i < NB; ++i) dq[i] = mma(kt[g][i], ds, dq[i]);
            }
        }
    };
    auto fetch = [&](int it) {
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            kr[g] = T::load(kfrom, it * KG + g);
            vr[g] = T::load(vfrom, it * KG + g);
        }
    };
    auto put = [&](char* to) {
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            T::store(to + 2 * g * T::kBytes, kr[g], tid);
            T::store(to + (2 * g + 1) * T::kBytes, vr[g], tid);
        }
    };
    const int turns = (stages + KG - 1) / KG;
    auto turn = [&](int it, char* here, char* there) {
        if (it + 1 < turns) fetch(it + 1);
        const int st = it * KG + grp;
        const char* at0 = here + 2 * grp * T::kBytes;
#pragma unroll
        for (int sub = 0; sub < R / 32; ++sub)
            if (st * R + sub * 32 < seen_hi)  // wave-uniform
                tile(at0 + sub * 32 * T::kRow, at0 + T::kBytes + sub * 32 * T::kRow, st * R + sub * 32);
        if (it + 1 < turns) put(there);
        __syncthreads();
    };
    if (turns > 0) {
        fetch(0);
        put(smem);
    }
    __syncthreads();
    for (int it = 0; it < turns; it += 2) {
        turn(it, smem, smem + kBuf);
        if (it + 1 < turns) turn(it + 1, smem + kBuf, smem);
    }
    if (KG == 2) {
        float* park = reinterpret_cast<float*>(smem) + (wave % W) * 64 * (NB * 32 + 3) + lane;
        if (grp == 1) {
            park[0] = off;
            if (X::kScaled) {
                park[64 * (NB * 32 + 1)] = gs.set() ? gs.x : INFINITY;
                park[64 * (NB * 32 + 2)] = gs.top;
            }
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    park[64 * (1 + 32 * i + r)] = dq[i][r];
                    park[64 * (17 + 32 * i + r)] = pk[i][r];
                }
        }
        __syncthreads();
        if (grp == 1) return;
        float f1 = 1.f, f2 = 1.f;
        if (X::kScaled) {  // the smaller of the two factors (one that was not set goes with sums of 0)
            const float x1 = gs.set() ? gs.x : INFINITY, x2 = park[64 * (NB * 32 + 1)], x = fminf(x1, x2);
            if (x1 != INFINITY) f1 = x / x1;
            if (x2 != INFINITY) f2 = x / x2;
            if (x != INFINITY) gs.x = x, gs.limit = 32768.f;
            gs.top = fmaxf(gs.top * f1, park[64 * (NB * 32 + 2)] * f2);
        }
        off = off * f1 + park[0] * f2;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dq[i][r] = dq[i][r] * f1 + park[64 * (1 + 32 * i + r)] * f2;
                pk[i][r] += park[64 * (17 + 32 * i + r)];
            }
    }
    off = sum_halves(off);
    const float unit = X::kScaled ? X::kUnprob / gs.x : 1.f;  // of dq and off
    if (X::kScaled && q0 < a.Tq) {
        // (the dK / dV kernel takes D corrected by off, which changes dS by off P at most)
        float most = gs.set() && in ? (gs.top + fabsf(off)) / gs.x : 0.f;
        if (!(most < INFINITY)) most = 0.f;  // a row whose gradient is not finite is no measure for the others
        most = max_wave(most);
        if (lane == 0) a.delta[delta_floats(a) + static_cast<long>(bh) * bounds_of_head(a) + (q0 >> 5)] = most;
    }
    if (qi >= a.Tq) return;
    if (hh == 0) a.delta[row] = delta + off * unit;
    E* drow = static_cast<E*>(a.dq) + b * a.sdq.b + qi * a.sdq.t + h * a.sdq.h;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            typename T::x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * g + e;
                v[e] = static_cast<E>(in ? fmaf(-off * X::kUnprob, pk[i][r], dq[i][r]) * (a.scale * unit) : 0.f);
            }
            const int c = 32 * i + 8 * g + 4 * hh;
            if (c < a.D) *reinterpret_cast<typename T::x4*>(drow + c) = v;
        }
}

// ---------------------------------------------------------------------------------------------
// Backward, keys: one workgroup = 128 keys of one key head; streams Q / dO of every query head
// that reads them.  Where that makes too few workgroups (few sequences, shared heads) the stages of
// all heads are cut into ranges (key_plan), one workgroup each (blockIdx.z): they leave fp32 sums in
// `parts` ([range][dK, dV][B][Hk][Tk][DP]) that attn_add_kernel adds in order.  (6 ragged sequences
// of up to 777, 16 heads on 4 of 128: 145 us in 168 workgroups, 57 + 9 us in ranges; with the exponents of
// half 63 + 9.)
template <class E, int DP, bool kDrop, bool kFine>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP == 64 && !kFine ? 2 : 1)))
attn_dkdv_kernel(AttnArgs a) {
    constexpr int R = kStage, NB = DP / 32;
    typedef Exponent<E> X;
    typedef Tile<E, DP, R> T;
    typedef typename T::x8 x8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int bh = shifted_head(a, a.Hk), b = bh / a.Hk, hk = bh % a.Hk, group = a.H / a.Hk;
    const int tile0 = blockIdx.y * 128;  // key tile 0 is seen by every query: longest first
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hh = lane >> 5;
    const Seq sq = sequence(a, b);
    const KeyPlan plan = key_plan(a, sq, tile0);
    const int z = blockIdx.z, first = plan.first, per = plan.per;
    if (z >= plan.ranges) return;
    const int key0 = __builtin_amdgcn_readfirstlane(tile0 + wave * 32), kj = key0 + n;
    const typename T::Lane at = T::lane_offsets(lane);
    x8 kf[DP / 16], vf[DP / 16];
    own_row<E, DP>(static_cast<const E*>(a.k) + b * a.sk.b + hk * a.sk.h + kj * a.sk.t, kj < sq.n, a.D, hh, kf);
    own_row<E, DP>(static_cast<const E*>(a.v) + b * a.sv.b + hk * a.sv.h + kj * a.sv.t, kj < sq.n, a.D, hh, vf);
    f32x16 dk[NB], dv[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) { dk[i] = f32x16{0}; dv[i] = f32x16{0}; }
    const float sc2 = a.scale * kLog2e;
    const unsigned step = kDrop ? step_of(a) : 0u;
    // half: dS times x, so that the bound of all queries that read this key head comes to [2^13, 2^14)
    float x = X::kScaled ? 0.f : 1.f, xup = kDrop ? a.up : 1.f;
    auto find_scale = [&]() {
        const long nb = bounds_of_head(a), all = nb * group;  // (the heads of a group are neighbours)
        const float* bounds = a.delta + delta_floats(a) + (static_cast<long>(b) * a.H + hk * group) * nb;
        float most = 0.f;
#pragma unroll 4
        for (long i = lane; i < all; i += 64) most = fmaxf(most, bounds[i]);
        most = max_wave(most);
        x = most > 0.f ? ldexpf(1.f, min(14 - __builtin_amdgcn_frexp_expf(most), 60)) : 1.f;
        xup *= x;
    };

    constexpr int kBuf = 2 * T::kBytes + 2 * R * 4;
    typename T::Regs qr, dr;
    float ls = 0.f, de = 0.f;
    const int it0 = static_cast<int>(static_cast<long>(per) * group * z / plan.ranges);
    const int it1 = static_cast<int>(static_cast<long>(per) * group * (z + 1) / plan.ranges);
    for (int g = 0; g < group; ++g) {
        const int h = hk * group + g;
        const int lo = first + max(0, it0 - g * per), hi = first + min(per, it1 - g * per);  // stages of this head
        if (lo >= hi) continue;
        const typename T::From qfrom = T::from(a.q, b * a.sq.b + h * a.sq.h, a.sq.t, sq.m, a.D, tid);
        const typename T::From dfrom = T::from(a.dout, b * a.sdo.b + h * a.sdo.h, a.sdo.t, sq.m, a.D, tid);
        const long rows = (static_cast<long>(b) * a.H + h) * a.Tq;
        const unsigned head = static_cast<unsigned>(a.first_head + b * a.H + h);
        auto fetch = [&](int st) {
            qr = T::load(qfrom, st);
            dr = T::load(dfrom, st);
            if (tid < R) {
                const int i = st * R + tid;
                ls = i < sq.m ? a.lse[rows + i] : -INFINITY;
                de = i < sq.m ? a.delta[rows + i] : 0.f;
            }
        };
        auto fill = [&](char* base) {
            T::store(base, qr, tid);
            T::store(base + T::kBytes, dr, tid);
            if (tid < R) {
                reinterpret_cast<float*>(base + 2 * T::kBytes)[tid] = ls == -INFINITY ? INFINITY : ls * kLog2e - X::kProb;
                reinterpret_cast<float*>(base + 2 * T::kBytes)[R + tid] = X::kScaled ? de * x : de;
            }
        };
        auto tile = [&](const char* Qs, const char* Ds, const float* lse2, const float* del, int qs0) {
            f32x16 s = {0}, dp = {0};
#pragma unroll
            for (int part = 0; part < DP / 64; ++part) {
                x8 f[4], e[4];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    f[ks] = T::row(Qs, at, 0, 4 * part + ks);
                    e[ks] = T::row(Ds, at, 0, 4 * part + ks);
                }
                reads_first();
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    s = mma(f[ks], kf[4 * part + ks], s);
                    dp = mma(e[ks], vf[4 * part + ks], dp);
                }
            }
            x8 qt[2][NB], dt[2][NB];
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    qt[g][i] = T::tr(Qs, at, 16 * g, i);
                    dt[g][i] = T::tr(Ds, at, 16 * g, i);
                }
            reads_first();
            unsigned w[4];
            if (kDrop) mask_bytes<false>(w, a.seed, head, step, qs0, key0, lane);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse2 + 8 * q + 4 * hh);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * q + e] = exp2_fast(fmaf(s[4 * q + e], sc2, -l4[e]));
            }
            if (qs0 + sq.off < key0 + 31) {  // wave-uniform: some query of the tile precedes some key
                keep_branch();
                const int lim = kj - sq.off - qs0 - 4 * hh;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (reg_row(r) < lim) s[r] = 0.f;
            }
            f32x16 pd = s;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(del + 8 * q + 4 * hh);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * q + e;
                    if (kDrop) {
                        const bool in = kept(w, r, a.limit);
                        pd[r] = in ? s[r] : 0.f;
                        dp[r] = s[r] * fmaf(dp[r], in ? xup : 0.f, -d4[e]);
                    } else if (X::kScaled) {
                        dp[r] = s[r] * fmaf(dp[r], xup, -d4[e]);
                    } else {
                        dp[r] = s[r] * (dp[r] - d4[e]);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const x8 p = pack8<E>(pd, 8 * k), ds = pack8<E>(dp, 8 * k);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    dv[i] = mma(p, dt[k][i], dv[i]);
                    dk[i] = mma(ds, qt[k][i], dk[i]);
                }
            }
            if (kFine) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const x8 p = rest8<E>(pd, 8 * k), ds = rest8<E>(dp, 8 * k);
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        dv[i] = mma(p, dt[k][i], dv[i]);
                        dk[i] = mma(ds, qt[k][i], dk[i]);
                    }
                }
            }
        };
        auto stage = [&](int st, char* here, char* there) {
            if (st + 1 < hi) fetch(st + 1);
            const float* lse2 = reinterpret_cast<const float*>(here + 2 * T::kBytes);
#pragma unroll
            for (int sub = 0; sub < R / 32; ++sub) {
                const int qs0 = st * R + sub * 32;
                // wave-uniform: every query of the tile precedes every key, or there is none
                if (qs0 + 31 + sq.off >= key0 && qs0 < sq.m)
                    tile(here + sub * 32 * T::kRow, here + T::kBytes + sub * 32 * T::kRow, lse2 + sub * 32,
                         lse2 + R + sub * 32, qs0);
            }
            if (st + 1 < hi) fill(there);
            __syncthreads();
        };
        fetch(lo);
        if (X::kScaled && x == 0.f) find_scale();  // (once, while the first stage is on its way)
        fill(smem);
        __syncthreads();
        for (int st = lo; st < hi; st += 2) {
            stage(st, smem, smem + kBuf);
            if (st + 1 < hi) stage(st + 1, smem + kBuf, smem);
        }
    }
    // register r of block i: key key0 + acc_row(r), column 32 i + n.  (The factor of what is kept
    // comes last: the probabilities are rounded without it, so that a probability of 1 stays exact.)
    const float up = (kDrop ? a.up : 1.f) * X::kUnprob;
    const float scale = X::kScaled ? a.scale * (X::kUnprob / (x > 0.f ? x : 1.f)) : a.scale;
    if (plan.ranges > 1) {
        const long heads = static_cast<long>(a.B) * a.Hk;
        float* pk = a.parts + ((2L * z * heads + bh) * a.Tk) * DP;
        float* pv = pk + heads * a.Tk * DP;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = key0 + acc_row(r, lane);
            if (j >= sq.n) continue;  // (not read)
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                pk[static_cast<long>(j) * DP + 32 * i + n] = dk[i][r] * scale;
                pv[static_cast<long>(j) * DP + 32 * i + n] = dv[i][r] * up;
            }
        }
        return;
    }
    E* dkb = static_cast<E*>(a.dk) + b * a.sdk.b + hk * a.sdk.h;
    E* dvb = static_cast<E*>(a.dv) + b * a.sdv.b + hk * a.sdv.h;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int j = key0 + acc_row(r, lane);
        if (j >= a.Tk) continue;
        const bool in = j < sq.n;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int c = 32 * i + n;
            if (c >= a.D) continue;
            dkb[j * a.sdk.t + c] = static_cast<E>(in ? dk[i][r] * scale : 0.f);
            dvb[j * a.sdv.t + c] = static_cast<E>(in ? dv[i][r] * up : 0.f);
        }
    }
}

// The ranges of attn_dkdv_kernel in order.  A thread takes four columns of a key's dK or dV.
template <class E, int DP>
__global__ void __launch_bounds__(256) attn_add_kernel(AttnArgs a) {
    const long heads = static_cast<long>(a.B) * a.Hk, one = heads * a.Tk * DP;
    const long at = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (at >= 2 * one) return;
    const bool v = at >= one;
    const long e = v ? at - one : at, row = e / DP;
    const int c = static_cast<int>(e % DP), j = static_cast<int>(row % a.Tk);
    const int b = static_cast<int>(row / a.Tk / a.Hk), hk = static_cast<int>(row / a.Tk % a.Hk);
    if (c >= a.D) return;
    const Seq sq = sequence(a, b);
    const int ranges = key_plan(a, sq, j & ~127).ranges;
    if (ranges == 1) return;  // written already
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (j < sq.n) {
        const float* p = a.parts + at;
        for (int z0 = 0; z0 < ranges; z0 += 4) {
            f32x4 x[4];
#pragma unroll
            for (int z = 0; z < 4; ++z)
                x[z] = z0 + z < ranges ? *reinterpret_cast<const f32x4*>(p + 2 * one * (z0 + z)) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int z = 0; z < 4; ++z) sum += x[z];
        }
    }
    typename Vec<E>::x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = static_cast<E>(sum[i]);
    const Strides& st = v ? a.sdv : a.sdk;
    *reinterpret_cast<typename Vec<E>::x4*>(static_cast<E*>(v ? a.dv : a.dk) + b * st.b + j * st.t + hk * st.h + c) = out;
}

// ---------------------------------------------------------------------------------------------
int set_lds(const void* fn, int bytes) {
    return hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess ? 0 : -20;
}

// Whether two waves share 32 queries (forward and dQ kernels): where the longest workgroup of a launch
// takes longer than its CUs' share of the whole.  At 64 columns, two halves to a CU, up to 512
// workgroups of 128 queries (1 x 4096, 12 heads: forward 75.6 -> 49.5 us, backward 167 -> 149; but 2 x
// 4096: 84.7 -> 86.8), or 1024 if there are lengths, which leave some of them empty (six of 0 .. 777, 16
// heads: 26.2 -> 20.9, 66 -> 60).  At 128, one half to a CU, below 256 (1 x 3624, 8 heads of 80: 88 -> 70,
// 231 -> 196; but 4 x 512, 16 heads, which makes 256: 19.8 -> 22.9, 54 -> 58).
bool halve_keys(const AttnArgs& a) {
    const long groups = static_cast<long>(a.B) * a.H * ((a.Tq + 127) / 128);
    const bool ragged = a.qlen != nullptr || a.klen != nullptr;
    return a.Tk > 4 * kStage && (a.D > 64 ? groups < 256 : groups <= (ragged ? 1024 : 512));
}

template <class E, int DP, bool kDrop, int KG>
int launch_fwd(const AttnArgs& a, hipStream_t s) {
    constexpr int lds = 4 * KG * Tile<E, DP, kStage>::kBytes;  // (the joint needs less)
    static_assert(KG == 1 || 2 * 64 * (DP / 2 + 2) * 4 <= lds, "room for the second waves' results");
    if (const int st = set_lds(reinterpret_cast<const void*>(attn_fwd_kernel<E, DP, kDrop, KG>), lds)) return st;
    hipLaunchKernelGGL((attn_fwd_kernel<E, DP, kDrop, KG>), dim3(a.B * a.H, (a.Tq + 128 / KG - 1) / (128 / KG)),
                       dim3(256), lds, s, a);
    return static_cast<int>(hipGetLastError());
}

template <class E, int DP, bool kDrop, int KG, bool kFine>
int launch_dq(const AttnArgs& a, hipStream_t s) {
    constexpr int ring = 4 * KG * Tile<E, DP, kStage>::kBytes, park = KG == 2 ? 2 * 64 * (DP + 3) * 4 : 0;
    constexpr int lds = ring > park ? ring : park;
    if (const int st = set_lds(reinterpret_cast<const void*>(attn_dq_kernel<E, DP, kDrop, KG, kFine>), lds)) return st;
    hipLaunchKernelGGL((attn_dq_kernel<E, DP, kDrop, KG, kFine>), dim3(a.B * a.H, (a.Tq + 128 / KG - 1) / (128 / KG)),
                       dim3(256), lds, s, a);
    return static_cast<int>(hipGetLastError());
}

// Workgroups that attn_few_kernel cuts the keys for (0: one per sequence and key head; -1: not the
// few-query form).
// More than one tile reads the keys once for each, the form for many queries once for each head, with
// one of four waves at work: several tiles pay against long caches where they are at most half as many
// as the heads that share a key head, or where there are few heads for the chip.  (8191 keys, 5 queries,
// 64 heads on 8 of 128, B 4: 48 us, 220 by head; 1024 keys, 32 queries, 32 heads on 4, B 2: 18, 24; but
// 48 heads on 12 of 64, B 8: 30, 21; 512 keys, 5 queries, 64 heads on 8 of 64, B 4: 14.7, 10.9.)
int few_tiles(const AttnArgs& a) { return (a.Tq * (a.H / a.Hk) + 31) / 32; }
int few_target(const AttnArgs& a) {
    const int group = a.H / a.Hk;
    if (a.limit != 0 || a.Tq > kFewQueries || group > kFewRows || a.Tq * group > kFewRows) return -1;
    const int tiles = few_tiles(a), target = kFewTarget / tiles;
    if (tiles > 1 && (a.Tk < 1024 || (2 * tiles > group && static_cast<long>(a.B) * a.H > 128))) return -1;
    return static_cast<long>(a.B) * a.Hk < target && a.Tk > 128 ? target : 0;
}
int few_workgroups(const AttnArgs& a) { return a.target + a.B * a.Hk; }  // at most
int padded_dim(int D) { return D <= 64 ? 64 : 128; }

template <class E, int DP, bool kTwice>
int launch_few(const AttnArgs& a, hipStream_t s) {
    constexpr int lds = 8 * Tile<E, DP, 32>::kBytes + 4 * 64 * 4;
    if (a.target != 0 && a.parts == nullptr) return -2;
    if (const int st = set_lds(reinterpret_cast<const void*>(attn_few_kernel<E, DP, kTwice>), lds)) return st;
    hipLaunchKernelGGL((attn_few_kernel<E, DP, kTwice>), dim3(few_workgroups(a), few_tiles(a)), dim3(256), lds, s, a);
    if (a.target != 0)
        hipLaunchKernelGGL((attn_join_kernel<E, DP>), dim3((a.B * a.H * a.Tq + 3) / 4), dim3(256), 0, s, a,
                           few_workgroups(a));
    return static_cast<int>(hipGetLastError());
}

// Query ranges of the dK / dV kernel at most: two rounds of workgroups if all sequences were of full
// length (the sums of the ranges cost a launch and their way through memory), no more than eight.
// (Three rounds: 814 instead of 717 us with 2 sequences of 4096, 16 heads on 4 of 128.)
int key_splits(const AttnArgs& a) {
    const long groups = static_cast<long>(a.B) * a.Hk * ((a.Tk + 127) / 128);
    const long most = static_cast<long>(a.H / a.Hk) * ((a.Tq + kStage - 1) / kStage) / least_range(a.D);
    const long want = ((a.D > 64 ? 512 : 1024) + groups - 1) / groups;
    const long n = want < most ? want : most;
    return static_cast<int>(n < 1 ? 1 : n > 8 ? 8 : n);
}
// Whether the backward pass undoes the rounding of P and dS: for short sequences (by the lengths of the call
// alone, so that a sequence has the same gradients whatever shares its launch).  Error of dQ and dK over that of
// rounding them: 1.0, without it 1.41 at any length.  It costs nothing where launches bound the time (8
// sequences of 64, 12 heads of 64: 18.5 us both ways) and up to half where they are many (256 of them: 88 -> 128
// us; 30 % for 128 sequences of 128 or 8 of 1024, where attention is more of a layer's time).
bool fine(const AttnArgs& a) { return a.Tq <= kStage && a.Tk <= kStage; }

template <class E, int DP, bool kDrop, bool kFine>
int launch_bwd(const AttnArgs& a, hipStream_t s) {
    constexpr int lds = 4 * Tile<E, DP, kStage>::kBytes + 4 * kStage * 4;
    if (const int st = !kFine && halve_keys(a) ? launch_dq<E, DP, kDrop, 2, false>(a, s) : launch_dq<E, DP, kDrop, 1, kFine>(a, s)) return st;
    if (const int st = set_lds(reinterpret_cast<const void*>(attn_dkdv_kernel<E, DP, kDrop, kFine>), lds)) return st;
    hipLaunchKernelGGL((attn_dkdv_kernel<E, DP, kDrop, kFine>), dim3(a.B * a.Hk, (a.Tk + 127) / 128, a.splits), dim3(256),
                       lds, s, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((attn_add_kernel<E, DP>),
                           dim3(static_cast<unsigned>((2L * a.B * a.Hk * a.Tk * DP / 4 + 255) / 256)), dim3(256), 0, s, a);
    return static_cast<int>(hipGetLastError());
}

template <class E, int DP>
int launch(const AttnArgs& a, int backward, hipStream_t s) {
    if (backward && fine(a)) return a.limit ? launch_bwd<E, DP, true, true>(a, s) : launch_bwd<E, DP, false, true>(a, s);
    if (backward) return a.limit ? launch_bwd<E, DP, true, false>(a, s) : launch_bwd<E, DP, false, false>(a, s);
    if (a.target >= 0) return a.Tq * (a.H / a.Hk) <= 16 ? launch_few<E, DP, true>(a, s) : launch_few<E, DP, false>(a, s);
    if (halve_keys(a)) return a.limit ? launch_fwd<E, DP, true, 2>(a, s) : launch_fwd<E, DP, false, 2>(a, s);
    return a.limit ? launch_fwd<E, DP, true, 1>(a, s) : launch_fwd<E, DP, false, 1>(a, s);
}

bool fits(const void* p, const Strides& st) {
    return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st.b % 8 == 0 && st.t % 8 == 0 &&
           st.h % 8 == 0 && st.t >= 0 && st.t < (1L << 24);
}

}  // namespace

extern "C" {

int nf_attention_args_size() { return static_cast<int>(sizeof(AttnArgs)); }

// floats of scratch that a forward call needs (args->parts)
long nf_attention_fwd_floats(const AttnArgs* args) {
    AttnArgs a = *args;
    if (a.Hk <= 0 || (a.target = few_target(a)) <= 0) return 0;
    return static_cast<long>(few_workgroups(a)) * a.Tq * (a.H / a.Hk) * (2 + padded_dim(a.D));
}

// ... and a backward call (args->delta)
long nf_attention_bwd_floats(const AttnArgs* args) {
    const AttnArgs& a = *args;
    if (a.Hk <= 0 || a.Tk <= 0) return 0;
    const int n = key_splits(a);
    return delta_floats(a) + bound_floats(a) + (n > 1 ? 2L * n * a.B * a.Hk * a.Tk * padded_dim(a.D) : 0);
}

// type: 1 bf16, 2 half.  backward 0: reads q, k, v and writes out, lse; 1: reads q, k, v, out,
// lse, dout and writes dq, dk, dv (delta: nf_attention_bwd_floats of scratch, 16-byte aligned).
int nf_attention(const AttnArgs* args, int type, int backward, hipStream_t s) {
    AttnArgs a = *args;
    if (a.B <= 0 || a.H <= 0 || a.Hk <= 0 || a.Tq <= 0 || a.Tk <= 0 || a.H % a.Hk != 0) return -1;
    if (a.D <= 0 || a.D > 128 || a.D % 8 != 0 || a.limit > 255u || !(a.scale > 0.f)) return -1;
    if (a.Tq > (1 << 22) || a.Tk > (1 << 22) || static_cast<long>(a.B) * a.H > (1 << 23)) return -3;
    if (!fits(a.q, a.sq) || !fits(a.k, a.sk) || !fits(a.v, a.sv) || !fits(a.out, a.so)) return -2;
    if (a.lse == nullptr) return -2;
    if (backward && (!fits(a.dout, a.sdo) || !fits(a.dq, a.sdq) || !fits(a.dk, a.sdk) ||
                     !fits(a.dv, a.sdv) || a.delta == nullptr))
        return -2;
    a.target = backward ? -1 : few_target(a);
    a.splits = backward ? key_splits(a) : 1;
    if (backward) a.parts = a.delta + delta_floats(a) + bound_floats(a);
    if (type == 1) return a.D <= 64 ? launch<bf16, 64>(a, backward, s) : launch<bf16, 128>(a, backward, s);
    if (type == 2) return a.D <= 64 ? launch<half, 64>(a, backward, s) : launch<half, 128>(a, backward, s);
    return -1;
}

}  // extern "C"
