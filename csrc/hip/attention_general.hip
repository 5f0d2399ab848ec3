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

struct Strides { long b, t, h; };  // elements between sequences, rows, heads

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;               // [B][H][Tq]
    const void* dout;
    void *dq, *dk, *dv;
    float* delta;             // [B][H][Tq], rowsum(dO * O): written by the dQ kernel
    const int *qlen, *klen;   // [B] or null
    const long* step_at;
    Strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
    unsigned long seed;
    unsigned long first_head; // number of the first head of the mask's counter
    int B, Tq, Tk, H, Hk, D, causal;
    float scale, up;
    unsigned limit, step;
};

// -- LDS tiles: 64 rows of DP columns --------------------------------------------------------
template <class E, int DP>
struct Tile {
    typedef typename Vec<E>::x8 x8;
    typedef typename Vec<E>::x4 x4;
    static constexpr int kBytes = kStage * DP * 2;
    static constexpr int kPieces = DP / 8;                 // 16-byte pieces of a row
    static constexpr int kPer = kStage * kPieces / 256;    // ... per thread (256 threads)
    struct Regs { uint4 v[kPer]; };

    // rows [r0, r0 + 64) of a matrix with `rows` rows and D columns; the rest reads as 0
    static __device__ __forceinline__ Regs load(const E* base, long ld, int r0, int rows, int D, int tid) {
        Regs t;
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
            const int idx = tid + 256 * p, r = r0 + idx / kPieces, c = (idx % kPieces) * 8;
            t.v[p] = make_uint4(0, 0, 0, 0);
            if (r < rows && c < D) t.v[p] = *reinterpret_cast<const uint4*>(base + r * ld + c);
        }
        return t;
    }
    static __device__ __forceinline__ void store(char* lds, const Regs& t, int tid) {
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
            const int idx = tid + 256 * p;
            *reinterpret_cast<uint4*>(lds + nfix::attn_off(DP, idx / kPieces, idx % kPieces)) = t.v[p];
        }
    }
    // operand fragment: row `row`, columns 16 ks + 8 (lane >> 5) .. + 7
    static __device__ __forceinline__ x8 row(const char* lds, int row, int ks, int hh) {
        return *reinterpret_cast<const x8*>(lds + nfix::attn_off(DP, row, 2 * ks + hh));
    }
    // 8 values tile[k0 + (j & 3) + 4 h + 8 (j >> 2)][x0 + (lane & 31)], h = lane >> 5: rows in the
    // order in which an accumulator hands them to the next MFMA
    static __device__ __forceinline__ x8 tr(const char* lds, int k0, int x0, int lane) {
        const int i = lane & 15;
        const int r = k0 + 4 * (lane >> 5) + (i >> 2), x = x0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
        const x4 lo = tr4(reinterpret_cast<const E*>(lds + nfix::attn_off(DP, r, x >> 3) + (x & 7) * 2));
        const x4 hi = tr4(reinterpret_cast<const E*>(lds + nfix::attn_off(DP, r + 8, x >> 3) + (x & 7) * 2));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

template <class E>
__device__ __forceinline__ typename Vec<E>::x8 pack8(const f32x16& v, int first) {
    typename Vec<E>::x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = static_cast<E>(v[first + j]);
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

__device__ __forceinline__ unsigned step_of(const AttnArgs& a) {
    return a.step_at != nullptr ? static_cast<unsigned>(*a.step_at) : a.step;
}

// ---------------------------------------------------------------------------------------------
// Forward: one workgroup = 128 queries (4 waves x 32) of one head; tiles of 64 keys, double-
// buffered in LDS.  grid = (sequence and head, tile): the tiles of a head land on one XCD, the
// long ones are dispatched first.
template <class E, int DP, bool kDrop>
__global__ void __launch_bounds__(256) attn_fwd_kernel(AttnArgs a) {
    typedef Tile<E, DP> T;
    typedef typename T::x8 x8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int bh = blockIdx.x, b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hk);
    const int tile0 = (gridDim.y - 1 - blockIdx.y) * 128;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hh = lane >> 5;
    const Seq sq = sequence(a, b);
    const E* qb = static_cast<const E*>(a.q) + b * a.sq.b + h * a.sq.h;
    const E* kb = static_cast<const E*>(a.k) + b * a.sk.b + hk * a.sk.h;
    const E* vb = static_cast<const E*>(a.v) + b * a.sv.b + hk * a.sv.h;
    const int q0 = tile0 + wave * 32, qi = q0 + n;
    const int stages = tile0 < sq.m ? (keys_seen(sq, min(tile0 + 127, sq.m - 1)) + kStage - 1) / kStage : 0;
    x8 qf[DP / 16];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        qf[ks] = {};
        const int c = ks * 16 + 8 * hh;
        if (qi < sq.m && c < a.D) qf[ks] = *reinterpret_cast<const x8*>(qb + qi * a.sq.t + c);
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = f32x16{0};
    float m = -INFINITY, l = 0.f;
    const float sc2 = a.scale * kLog2e;
    // keys that the wave's first and last query see, and this lane's
    const int seen_lo = keys_seen(sq, q0), seen = keys_seen(sq, qi);
    const int seen_hi = q0 < sq.m ? keys_seen(sq, q0 + 31) : 0;
    const unsigned step = kDrop ? step_of(a) : 0u, head = static_cast<unsigned>(a.first_head + bh);

    typename T::Regs kr, vr;
    if (stages > 0) {
        kr = T::load(kb, a.sk.t, 0, sq.n, a.D, tid);
        vr = T::load(vb, a.sv.t, 0, sq.n, a.D, tid);
        T::store(smem, kr, tid);
        T::store(smem + 2 * T::kBytes, vr, tid);
    }
    __syncthreads();
    for (int st = 0; st < stages; ++st) {
        const char* Ks = smem + (st & 1) * T::kBytes;
        const char* Vs = smem + (2 + (st & 1)) * T::kBytes;
        if (st + 1 < stages) {
            kr = T::load(kb, a.sk.t, (st + 1) * kStage, sq.n, a.D, tid);
            vr = T::load(vb, a.sv.t, (st + 1) * kStage, sq.n, a.D, tid);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int key0 = st * kStage + sub * 32;
            if (key0 >= seen_hi) continue;  // wave-uniform: nothing visible in this tile
            f32x16 s = {0};
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) s = mma(T::row(Ks, sub * 32 + n, ks, hh), qf[ks], s);
            if (key0 + 32 > seen_lo) {      // wave-uniform: some pair of the tile is not visible
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (key0 + acc_row(r, lane) >= seen) s[r] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (__any(mx > m)) {  // the running maximum rarely moves after the first tiles
                const float mn = fmaxf(m, mx);
                const float ref = mn == -INFINITY ? 0.f : mn;
                const float alpha = exp2_fast((m - ref) * sc2);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
            }
            const float msc = m == -INFINITY ? 0.f : m * sc2;
            float rs = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = exp2_fast(fmaf(s[r], sc2, -msc));
                rs += s[r];
            }
            l += rs;
            if (kDrop) {  // the sum is of all probabilities, what is dropped leaves the product
                unsigned w[4];
                mask_bytes<true>(w, a.seed, head, step, key0, q0, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!kept(w, r, a.limit)) s[r] = 0.f;
            }
            const x8 p0 = pack8<E>(s, 0), p1 = pack8<E>(s, 8);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                o[i] = mma(T::tr(Vs, sub * 32, 32 * i, lane), p0, o[i]);
                o[i] = mma(T::tr(Vs, sub * 32 + 16, 32 * i, lane), p1, o[i]);
            }
        }
        if (st + 1 < stages) {
            T::store(smem + ((st + 1) & 1) * T::kBytes, kr, tid);
            T::store(smem + (2 + ((st + 1) & 1)) * T::kBytes, vr, tid);
        }
        __syncthreads();
    }
    if (qi >= a.Tq) return;
    l += __shfl_xor(l, 32, 64);
    const bool some = qi < sq.m && l > 0.f;
    const float inv = some || l != l ? (kDrop ? a.up : 1.f) / l : 0.f;
    E* orow = static_cast<E*>(a.out) + b * a.so.b + qi * a.so.t + h * a.so.h;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            typename T::x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<E>(qi < sq.m ? o[i][4 * g + e] * inv : 0.f);
            const int c = 32 * i + 8 * g + 4 * hh;
            if (c < a.D) *reinterpret_cast<typename T::x4*>(orow + c) = v;
        }
    if (hh == 0)
        a.lse[static_cast<long>(bh) * a.Tq + qi] =
            qi < sq.m && (some || l != l) ? m * a.scale + kLn2 * __builtin_amdgcn_logf(l) : -INFINITY;
}

// ---------------------------------------------------------------------------------------------
// Backward, queries: one workgroup = 128 queries; streams K / V.  Also leaves D = rowsum(dO * O)
// for the dK / dV kernel that follows.
template <class E, int DP, bool kDrop>
__global__ void __launch_bounds__(256) attn_dq_kernel(AttnArgs a) {
    typedef Tile<E, DP> T;
    typedef typename T::x8 x8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int bh = blockIdx.x, b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hk);
    const int tile0 = (gridDim.y - 1 - blockIdx.y) * 128;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hh = lane >> 5;
    const Seq sq = sequence(a, b);
    const E* qb = static_cast<const E*>(a.q) + b * a.sq.b + h * a.sq.h;
    const E* kb = static_cast<const E*>(a.k) + b * a.sk.b + hk * a.sk.h;
    const E* vb = static_cast<const E*>(a.v) + b * a.sv.b + hk * a.sv.h;
    const E* ob = static_cast<const E*>(a.out) + b * a.so.b + h * a.so.h;
    const E* dob = static_cast<const E*>(a.dout) + b * a.sdo.b + h * a.sdo.h;
    const int q0 = tile0 + wave * 32, qi = q0 + n;
    const int stages = tile0 < sq.m ? (keys_seen(sq, min(tile0 + 127, sq.m - 1)) + kStage - 1) / kStage : 0;
    x8 qf[DP / 16], df[DP / 16];
    float delta = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        qf[ks] = {};
        df[ks] = {};
        const int c = ks * 16 + 8 * hh;
        if (qi < sq.m && c < a.D) {
            qf[ks] = *reinterpret_cast<const x8*>(qb + qi * a.sq.t + c);
            df[ks] = *reinterpret_cast<const x8*>(dob + qi * a.sdo.t + c);
            const x8 of = *reinterpret_cast<const x8*>(ob + qi * a.so.t + c);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                delta = fmaf(static_cast<float>(df[ks][j]), static_cast<float>(of[j]), delta);
        }
    }
    delta += __shfl_xor(delta, 32, 64);
    const long at = static_cast<long>(bh) * a.Tq + qi;
    // a row that sees no key has lse -inf: +inf makes its probabilities 0
    float lse2 = INFINITY;
    if (qi < sq.m) {
        const float v = a.lse[at];
        lse2 = v == -INFINITY ? INFINITY : v * kLog2e;
    }
    if (qi < a.Tq && hh == 0) a.delta[at] = delta;
    f32x16 dq[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dq[i] = f32x16{0};
    const float sc2 = a.scale * kLog2e;
    const int seen_lo = keys_seen(sq, q0), seen = keys_seen(sq, qi);
    const int seen_hi = q0 < sq.m ? keys_seen(sq, q0 + 31) : 0;
    const unsigned step = kDrop ? step_of(a) : 0u, head = static_cast<unsigned>(a.first_head + bh);

    typename T::Regs kr, vr;
    if (stages > 0) {
        kr = T::load(kb, a.sk.t, 0, sq.n, a.D, tid);
        vr = T::load(vb, a.sv.t, 0, sq.n, a.D, tid);
        T::store(smem, kr, tid);
        T::store(smem + 2 * T::kBytes, vr, tid);
    }
    __syncthreads();
    for (int st = 0; st < stages; ++st) {
        const char* Ks = smem + (st & 1) * T::kBytes;
        const char* Vs = smem + (2 + (st & 1)) * T::kBytes;
        if (st + 1 < stages) {
            kr = T::load(kb, a.sk.t, (st + 1) * kStage, sq.n, a.D, tid);
            vr = T::load(vb, a.sv.t, (st + 1) * kStage, sq.n, a.D, tid);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int key0 = st * kStage + sub * 32;
            if (key0 >= seen_hi) continue;
            f32x16 s = {0}, dp = {0};
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                s = mma(T::row(Ks, sub * 32 + n, ks, hh), qf[ks], s);
                dp = mma(T::row(Vs, sub * 32 + n, ks, hh), df[ks], dp);
            }
            unsigned w[4];
            if (kDrop) mask_bytes<true>(w, a.seed, head, step, key0, q0, lane);
            const bool edge = key0 + 32 > seen_lo;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = exp2_fast(fmaf(s[r], sc2, -lse2));
                float d = dp[r];
                if (kDrop) d = kept(w, r, a.limit) ? d * a.up : 0.f;
                s[r] = p * (d - delta);
            }
            if (edge) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (key0 + acc_row(r, lane) >= seen) s[r] = 0.f;
            }
            const x8 s0 = pack8<E>(s, 0), s1 = pack8<E>(s, 8);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                dq[i] = mma(T::tr(Ks, sub * 32, 32 * i, lane), s0, dq[i]);
                dq[i] = mma(T::tr(Ks, sub * 32 + 16, 32 * i, lane), s1, dq[i]);
            }
        }
        if (st + 1 < stages) {
            T::store(smem + ((st + 1) & 1) * T::kBytes, kr, tid);
            T::store(smem + (2 + ((st + 1) & 1)) * T::kBytes, vr, tid);
        }
        __syncthreads();
    }
    if (qi >= a.Tq) return;
    E* drow = static_cast<E*>(a.dq) + b * a.sdq.b + qi * a.sdq.t + h * a.sdq.h;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            typename T::x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<E>(qi < sq.m ? dq[i][4 * g + e] * a.scale : 0.f);
            const int c = 32 * i + 8 * g + 4 * hh;
            if (c < a.D) *reinterpret_cast<typename T::x4*>(drow + c) = v;
        }
}

// ---------------------------------------------------------------------------------------------
// Backward, keys: one workgroup = 128 keys of one key head; streams Q / dO of every query head
// that reads them.
template <class E, int DP, bool kDrop>
__global__ void __launch_bounds__(256) attn_dkdv_kernel(AttnArgs a) {
    typedef Tile<E, DP> T;
    typedef typename T::x8 x8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int bh = blockIdx.x, b = bh / a.Hk, hk = bh % a.Hk, group = a.H / a.Hk;
    const int tile0 = blockIdx.y * 128;  // key tile 0 is seen by every query: longest first
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hh = lane >> 5;
    const Seq sq = sequence(a, b);
    const E* kb = static_cast<const E*>(a.k) + b * a.sk.b + hk * a.sk.h;
    const E* vb = static_cast<const E*>(a.v) + b * a.sv.b + hk * a.sv.h;
    const int key0 = tile0 + wave * 32, kj = key0 + n;
    x8 kf[DP / 16], vf[DP / 16];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        kf[ks] = {};
        vf[ks] = {};
        const int c = ks * 16 + 8 * hh;
        if (kj < sq.n && c < a.D) {
            kf[ks] = *reinterpret_cast<const x8*>(kb + kj * a.sk.t + c);
            vf[ks] = *reinterpret_cast<const x8*>(vb + kj * a.sv.t + c);
        }
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) { dk[i] = f32x16{0}; dv[i] = f32x16{0}; }
    const float sc2 = a.scale * kLog2e;
    const unsigned step = kDrop ? step_of(a) : 0u;
    // query i sees key j from i >= j - off on
    const int first = tile0 < sq.n ? max(0, a.causal ? tile0 - sq.off : 0) / kStage : 0;
    const int stages = tile0 < sq.n ? (sq.m + kStage - 1) / kStage : 0;
    const int per_head = max(0, stages - first), total = per_head * group;

    constexpr int kBuf = 2 * T::kBytes + 2 * kStage * 4;
    typename T::Regs qr, dr;
    float ls = 0.f, de = 0.f;
    auto fetch = [&](int it) {
        const int h = hk * group + it / per_head, r0 = (first + it % per_head) * kStage;
        qr = T::load(static_cast<const E*>(a.q) + b * a.sq.b + h * a.sq.h, a.sq.t, r0, sq.m, a.D, tid);
        dr = T::load(static_cast<const E*>(a.dout) + b * a.sdo.b + h * a.sdo.h, a.sdo.t, r0, sq.m, a.D, tid);
        if (tid < kStage) {
            const long at = (static_cast<long>(b) * a.H + h) * a.Tq + r0 + tid;
            const bool in = r0 + tid < sq.m;
            ls = in ? a.lse[at] : -INFINITY;
            ls = ls == -INFINITY ? INFINITY : ls * kLog2e;
            de = in ? a.delta[at] : 0.f;
        }
    };
    auto fill = [&](char* base) {
        T::store(base, qr, tid);
        T::store(base + T::kBytes, dr, tid);
        if (tid < kStage) {
            reinterpret_cast<float*>(base + 2 * T::kBytes)[tid] = ls;
            reinterpret_cast<float*>(base + 2 * T::kBytes)[kStage + tid] = de;
        }
    };
    if (total > 0) {
        fetch(0);
        fill(smem);
    }
    __syncthreads();
    for (int it = 0; it < total; ++it) {
        const char* Qs = smem + (it & 1) * kBuf;
        const char* Ds = Qs + T::kBytes;
        const float* lse2 = reinterpret_cast<const float*>(Qs + 2 * T::kBytes);
        const float* del = lse2 + kStage;
        const int st = first + it % per_head;
        const unsigned head = static_cast<unsigned>(a.first_head + b * a.H + hk * group + it / per_head);
        if (it + 1 < total) fetch(it + 1);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int qs0 = st * kStage + sub * 32;
            // wave-uniform: every query of the tile precedes every key, or there is none
            if (qs0 + 31 + sq.off < key0 || qs0 >= sq.m) continue;
            f32x16 s = {0}, dp = {0};
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                s = mma(T::row(Qs, sub * 32 + n, ks, hh), kf[ks], s);
                dp = mma(T::row(Ds, sub * 32 + n, ks, hh), vf[ks], dp);
            }
            unsigned w[4];
            if (kDrop) mask_bytes<false>(w, a.seed, head, step, qs0, key0, lane);
            const bool edge = qs0 + sq.off < key0 + 31;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 l4 = *reinterpret_cast<const float4*>(lse2 + sub * 32 + 8 * g + 4 * hh);
                const float4 d4 = *reinterpret_cast<const float4*>(del + sub * 32 + 8 * g + 4 * hh);
                const float lv[4] = {l4.x, l4.y, l4.z, l4.w}, dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * g + e;
                    float p = exp2_fast(fmaf(s[r], sc2, -lv[e])), d = dp[r];
                    if (edge && kj > qs0 + 8 * g + 4 * hh + e + sq.off) p = 0.f;
                    const bool in = !kDrop || kept(w, r, a.limit);
                    if (kDrop) d = in ? d * a.up : 0.f;
                    s[r] = in ? p : 0.f;
                    dp[r] = p * (d - dl[e]);
                }
            }
            const x8 p0 = pack8<E>(s, 0), p1 = pack8<E>(s, 8);
            const x8 s0 = pack8<E>(dp, 0), s1 = pack8<E>(dp, 8);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                dv[i] = mma(p0, T::tr(Ds, sub * 32, 32 * i, lane), dv[i]);
                dv[i] = mma(p1, T::tr(Ds, sub * 32 + 16, 32 * i, lane), dv[i]);
                dk[i] = mma(s0, T::tr(Qs, sub * 32, 32 * i, lane), dk[i]);
                dk[i] = mma(s1, T::tr(Qs, sub * 32 + 16, 32 * i, lane), dk[i]);
            }
        }
        if (it + 1 < total) fill(smem + ((it + 1) & 1) * kBuf);
        __syncthreads();
    }
    // register r of block i: key key0 + acc_row(r), column 32 i + n
    E* dkb = static_cast<E*>(a.dk) + b * a.sdk.b + hk * a.sdk.h;
    E* dvb = static_cast<E*>(a.dv) + b * a.sdv.b + hk * a.sdv.h;
    const float up = kDrop ? a.up : 1.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int j = key0 + acc_row(r, lane);
        if (j >= a.Tk) continue;
        const bool in = j < sq.n;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
            const int c = 32 * i + n;
            if (c >= a.D) continue;
            dkb[j * a.sdk.t + c] = static_cast<E>(in ? dk[i][r] * a.scale : 0.f);
            dvb[j * a.sdv.t + c] = static_cast<E>(in ? dv[i][r] * up : 0.f);
        }
    }
}

// ---------------------------------------------------------------------------------------------
int set_lds(const void* fn, int bytes) {
    return hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess ? 0 : -20;
}

template <class E, int DP, bool kDrop>
int launch_fwd(const AttnArgs& a, hipStream_t s) {
    constexpr int lds = 4 * Tile<E, DP>::kBytes;
    if (const int st = set_lds(reinterpret_cast<const void*>(attn_fwd_kernel<E, DP, kDrop>), lds)) return st;
    hipLaunchKernelGGL((attn_fwd_kernel<E, DP, kDrop>), dim3(a.B * a.H, (a.Tq + 127) / 128), dim3(256), lds, s, a);
    return static_cast<int>(hipGetLastError());
}

template <class E, int DP, bool kDrop>
int launch_bwd(const AttnArgs& a, hipStream_t s) {
    constexpr int lds = 4 * Tile<E, DP>::kBytes, lds2 = lds + 4 * kStage * 4;
    if (const int st = set_lds(reinterpret_cast<const void*>(attn_dq_kernel<E, DP, kDrop>), lds)) return st;
    if (const int st = set_lds(reinterpret_cast<const void*>(attn_dkdv_kernel<E, DP, kDrop>), lds2)) return st;
    hipLaunchKernelGGL((attn_dq_kernel<E, DP, kDrop>), dim3(a.B * a.H, (a.Tq + 127) / 128), dim3(256), lds, s, a);
    hipLaunchKernelGGL((attn_dkdv_kernel<E, DP, kDrop>), dim3(a.B * a.Hk, (a.Tk + 127) / 128), dim3(256), lds2, s, a);
    return static_cast<int>(hipGetLastError());
}

template <class E, int DP>
int launch(const AttnArgs& a, int backward, hipStream_t s) {
    if (backward) return a.limit ? launch_bwd<E, DP, true>(a, s) : launch_bwd<E, DP, false>(a, s);
    return a.limit ? launch_fwd<E, DP, true>(a, s) : launch_fwd<E, DP, false>(a, s);
}

bool fits(const void* p, const Strides& st) {
    return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st.b % 8 == 0 && st.t % 8 == 0 &&
           st.h % 8 == 0;
}

}  // namespace

extern "C" {

int nf_attention_args_size() { return static_cast<int>(sizeof(AttnArgs)); }

// type: 1 bf16, 2 half.  backward 0: reads q, k, v and writes out, lse; 1: reads q, k, v, out,
// lse, dout and writes dq, dk, dv (delta: B H Tq floats of scratch).
int nf_attention(const AttnArgs* args, int type, int backward, hipStream_t s) {
    const AttnArgs& a = *args;
    if (a.B <= 0 || a.H <= 0 || a.Hk <= 0 || a.Tq <= 0 || a.Tk <= 0 || a.H % a.Hk != 0) return -1;
    if (a.D <= 0 || a.D > 128 || a.D % 8 != 0 || a.limit > 255u || !(a.scale > 0.f)) return -1;
    if (a.Tq > (1 << 22) || a.Tk > (1 << 22) || static_cast<long>(a.B) * a.H > (1 << 23)) return -3;
    if (!fits(a.q, a.sq) || !fits(a.k, a.sk) || !fits(a.v, a.sv) || !fits(a.out, a.so)) return -2;
    if (a.lse == nullptr) return -2;
    if (backward && (!fits(a.dout, a.sdo) || !fits(a.dq, a.sdq) || !fits(a.dk, a.sdk) ||
                     !fits(a.dv, a.sdv) || a.delta == nullptr))
        return -2;
    if (type == 1) return a.D <= 64 ? launch<bf16, 64>(a, backward, s) : launch<bf16, 128>(a, backward, s);
    if (type == 2) return a.D <= 64 ? launch<half, 64>(a, backward, s) : launch<half, 128>(a, backward, s);
    return -1;
}

}  // extern "C"
