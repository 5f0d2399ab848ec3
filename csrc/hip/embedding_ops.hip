// Embedding lookup with scaling, positions and dropout, and its gradient by sorted tokens,
// for gfx950.  float, bf16 and half tables; sums in fp32.
//
//   x[r]    = drop(scale * W[t_r] + P[r mod T])
//   dW[v]   = scale * sum over {r : t_r = v, v != padding} of drop'(dx[r])
//   dP[t]   = sum over b of drop'(dx[b T + t])
//
// A token outside [0, V) looks up a row of zeros and has no gradient.
//
// Bound by memory: 32768 tokens of a 50257 x 768 bf16 table with positions and dropout take 21 us
// forward (4.8 TB/s); backward 21 us for the order, 38 us for the sums (dx read for the table and for
// the positions, 4.7 TB/s) and 7 us for the join of frequent tokens.

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

// ---------------------------------------------------------------------------------------------
// Order by token.  A token without a gradient (outside the table, padding) has the key V.
__device__ __forceinline__ unsigned key_of(const long* tokens, long i, unsigned V, long padding) {
    const long t = tokens[i];
    return t < 0 || t >= static_cast<long>(V) || t == padding ? V : static_cast<unsigned>(t);
}

// Few tokens, one launch: the place of row i is the number of rows with a smaller key, or the
// same key and a smaller index.  A workgroup holds all keys in LDS and places 16 rows: lane l has
// row l % 16 and looks at every fourth block of 16 keys of its wave, four per LDS read and two vector
// instructions each.  (Bound by these; 4000 rows: 5.2 us, with 64 rows per workgroup, a quarter as
// many of them, 10.2.)
constexpr int kRankWaves = 16, kRankRows = 8192;

__global__ void __launch_bounds__(64 * kRankWaves) rank_kernel(const long* tokens, unsigned V, long padding,
                                                               unsigned* key, unsigned* order, int R) {
    __shared__ __attribute__((aligned(16))) unsigned keys[kRankRows];
    __shared__ unsigned count[kRankWaves][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 15, i0 = blockIdx.x * 16, i = i0 + row, padded = (R + 63) & ~63;
    // (behind the last row: keys that no row is behind)
#pragma unroll 8
    for (int j = threadIdx.x; j < padded; j += 64 * kRankWaves)
        keys[j] = j < R ? key_of(tokens, j, V, padding) : 0xFFFFFFFFu;
    __syncthreads();
    const unsigned mine = keys[i];  // (i < padded)
    // equal keys count in the blocks before the row's own, and in that (a key per wave) before the row
    unsigned n = lane < 16 && wave < row && keys[i0 + wave] == mine;
    for (int j0 = wave * 64 + (lane & 48); j0 < padded; j0 += 64 * kRankWaves) {
        const unsigned limit = mine + (j0 < i0);  // count keys < limit (mine <= V < 2^31)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const uint4 k = *reinterpret_cast<const uint4*>(&keys[j0 + j]);
            n += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
        }
    }
    n += __shfl_xor(n, 16, 64);
    n += __shfl_xor(n, 32, 64);
    if (lane < 16) count[wave][lane] = n;
    __syncthreads();
    if (threadIdx.x >= 16 || i >= R) return;
    unsigned place = 0;
#pragma unroll
    for (int w = 0; w < kRankWaves; ++w) place += count[w][lane];
    key[place] = mine;
    order[place] = static_cast<unsigned>(i);
}

// Many tokens: stable counting sort by 8 bits at a time, lowest first.  One launch counts the
// lowest digits of every tile; then one launch for each digit, in which every workgroup finds its
// own first places from all counts, moves its tile and counts the next digit of what it moved in
// the tiles where that lands (whole numbers, so the order of these atomics changes nothing).  A tile
// is 256 * rounds keys, four waves with 64 * rounds consecutive ones each; with at most 128 tiles
// the counts are 128 rows of 1 KiB that every workgroup can read for itself, which is cheaper than
// a launch for their running sums.
constexpr int kDigits = 256, kMaxTiles = 128, kMaxPasses = 4;

__device__ __forceinline__ unsigned tile_key(const long* tokens, const unsigned* from, long i, unsigned V,
                                             long padding) {
    return tokens != nullptr ? key_of(tokens, i, V, padding) : from[i];
}

// count[tile][digit] of the lowest digit; the counts of `later` digits are set to 0.
__global__ void __launch_bounds__(256) digit_count_kernel(const long* tokens, unsigned V, long padding,
                                                          unsigned* count, long R, int rounds, int later) {
    __shared__ unsigned hist[kDigits];
    hist[threadIdx.x] = 0;
    for (int p = 1; p <= later; ++p) count[(p * kMaxTiles + blockIdx.x) * kDigits + threadIdx.x] = 0;
    __syncthreads();
    const long i0 = static_cast<long>(blockIdx.x) * rounds * 256;
#pragma unroll 4
    for (int k = 0; k < rounds; ++k) {
        const long i = i0 + k * 256 + threadIdx.x;
        if (i < R) atomicAdd(&hist[key_of(tokens, i, V, padding) & 255u], 1u);
    }
    __syncthreads();
    count[blockIdx.x * kDigits + threadIdx.x] = hist[threadIdx.x];
}

// Within a wave the keys go 64 at a time: lanes with the same digit are found by eight ballots, a
// lane's rank is the number of them before it.
__global__ void __launch_bounds__(256) digit_move_kernel(const long* tokens, const unsigned* from,
                                                         const unsigned* from_order, unsigned V,
                                                         long padding, const unsigned* count,
                                                         unsigned* next_count, unsigned* key,
                                                         unsigned* order, long R, int rounds, int shift) {
    __shared__ unsigned next[4][kDigits];
    __shared__ unsigned sums[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long i0 = (static_cast<long>(blockIdx.x) * 4 + wave) * rounds * 64;
#pragma unroll
    for (int w = 0; w < 4; ++w) next[w][threadIdx.x] = 0;
    __syncthreads();
    for (int r = 0; r < rounds; ++r) {
        const long i = i0 + r * 64 + lane;
        if (i < R) atomicAdd(&next[wave][(tile_key(tokens, from, i, V, padding) >> shift) & 255u], 1u);
    }
    // thread d: keys with digit d in the tiles before this one, and in all
    unsigned before = 0, all = 0;
    const int tiles = gridDim.x, mine = blockIdx.x;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        unsigned n[32];  // (all in flight: the loop's time is that of its loads one after another)
#pragma unroll
        for (int t = 0; t < 32; ++t) n[t] = count[min(t0 + t, tiles - 1) * kDigits + threadIdx.x];
#pragma unroll
        for (int t = 0; t < 32; ++t) {
            before += t0 + t < mine ? n[t] : 0u;
            all += t0 + t < tiles ? n[t] : 0u;
        }
    }
    unsigned x = all;  // running sum over the digits
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const unsigned y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
    }
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    unsigned at = before + x - all;
    for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
    for (int w = 0; w < 4; ++w) {  // every wave's first place of digit threadIdx.x
        const unsigned n = next[w][threadIdx.x];
        next[w][threadIdx.x] = at;
        at += n;
    }
    __syncthreads();
    for (int r = 0; r < rounds; ++r) {
        const long i = i0 + r * 64 + lane;
        const bool in = i < R;
        const unsigned k = in ? tile_key(tokens, from, i, V, padding) : 0u, d = (k >> shift) & 255u;
        const unsigned o = in && from_order != nullptr ? from_order[i] : static_cast<unsigned>(i);
        unsigned long same = __ballot(in);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const unsigned long ones = __ballot((d >> b) & 1u);
            same &= (d >> b) & 1u ? ones : ~ones;
        }
        const unsigned long below = same & ((1UL << lane) - 1UL);
        // (the LDS operations of a wave complete in order: every lane reads before the first lane
        // of each digit writes)
        const unsigned first = in ? next[wave][d] : 0u;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (in && below == 0) next[wave][d] = first + static_cast<unsigned>(__popcll(same));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (in) {
            const unsigned place = first + static_cast<unsigned>(__popcll(below));
            key[place] = k;
            order[place] = o;
            if (next_count != nullptr)
                atomicAdd(&next_count[place / (256u * rounds) * kDigits + ((k >> shift >> 8) & 255u)], 1u);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Gradients.  The sorted positions are cut into chunks of `chunk`; a wave sums one chunk over 512
// columns.  A run of equal tokens that lies within the chunk goes straight to its row; of a run
// that goes on, the chunk's part goes to head[chunk] (it began before) or tail[chunk] (it begins
// here), and the join kernel adds tail[chunk] + head[chunk + 1] + ... in a fixed order.  So a
// frequent token costs as many rows per wave as any other.
//
// The same launch holds the waves of the position gradient (one per position and 512 columns,
// summing over the sequences) and the workgroups that zero the rows of absent tokens (64 rows
// each, present ones found by a search in the sorted keys), so that every byte of the gradient is
// written once.
constexpr int kMaxChunk = 32;

struct BwdArgs {
    const unsigned *key, *order;
    const void* dx;
    void *dw, *dp;
    float *head, *tail;   // [chunks][C]
    long B, T, V, C;
    int R, chunk, chunks, slabs, accumulate;
    float scale;
    unsigned sum_blocks, pos_blocks;  // workgroups of the first two kinds
    DropRows d;
};

__device__ __forceinline__ void add8(float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] += b[i];
}

template <class G>
__device__ __forceinline__ void write_row(const BwdArgs& a, unsigned k, long c, int n, float (&acc)[8]) {
    G* row = static_cast<G*>(a.dw) + static_cast<long>(k) * a.C + c;
    float old[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (a.accumulate) load_unit(row, n, old);
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = fmaf(acc[q], a.scale, old[q]);
    store_unit(row, n, acc);
}

template <class T, class G>
__device__ __forceinline__ void sum_chunk(const BwdArgs& a, long w, int lane) {
    const int ch = static_cast<int>(w / a.slabs);
    if (ch >= a.chunks) return;
    const int p0 = ch * a.chunk, len = min(a.chunk, a.R - p0);
    // lane l holds key and row of position p0 - 1 + l (one before, one behind the chunk)
    const int p = p0 - 1 + lane;
    const bool there = p >= 0 && p < a.R && lane <= len + 1;
    const int kv = there ? static_cast<int>(a.key[p]) : -1, ov = there ? static_cast<int>(a.order[p]) : -1;
    const long c = (w % a.slabs) * 512 + lane * 8;
    const int n = a.C - c >= 8 ? 8 : static_cast<int>(a.C - c);  // <= 0: no columns
    const unsigned step = drop_step(a.d);
    const T* dx = static_cast<const T*>(a.dx);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    bool head = __builtin_amdgcn_readlane(kv, 0) == __builtin_amdgcn_readlane(kv, 1);
    constexpr int kBatch = 4;  // rows in flight
    for (int j0 = 0; j0 < len; j0 += kBatch) {
        float f[kBatch][8];
        long row[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            row[q] = j0 + q < len ? __builtin_amdgcn_readlane(ov, 1 + j0 + q) : -1;
            // (out of range: an order that is not of these tokens)
            const bool ok = row[q] >= 0 && row[q] < a.R && n > 0;
            if (ok) load_unit(dx + row[q] * a.C + c, n, f[q]);
            if (!ok) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[q][i] = 0.f;
            }
        }
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            if (j0 + q >= len) break;
            const int k = __builtin_amdgcn_readlane(kv, 1 + j0 + q), after = __builtin_amdgcn_readlane(kv, 2 + j0 + q);
            if (a.d.limit != 0 && row[q] >= 0) drop8(a.d, step, a.d.first + row[q] * a.C + c, f[q]);
            add8(acc, f[q]);
            const bool last = j0 + q + 1 == len;
            if (k == after && !last) continue;
            const bool known = k >= 0 && static_cast<unsigned>(k) < static_cast<unsigned>(a.V);
            if (known && n > 0) {
                if (head) store_unit(a.head + static_cast<long>(ch) * a.C + c, n, acc);
                else if (k == after) store_unit(a.tail + static_cast<long>(ch) * a.C + c, n, acc);
                else write_row<G>(a, static_cast<unsigned>(k), c, n, acc);
            }
            head = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = 0.f;
        }
    }
}

template <class T, class G>
__device__ __forceinline__ void sum_position(const BwdArgs& a, long w, int lane) {
    const long t = w / a.slabs, c = (w % a.slabs) * 512 + lane * 8;
    if (t >= a.T || c >= a.C) return;
    const int n = a.C - c >= 8 ? 8 : static_cast<int>(a.C - c);
    const unsigned step = drop_step(a.d);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (long b = 0; b < a.B; ++b) {
        const long e = (b * a.T + t) * a.C + c;
        float f[8];
        load_unit(static_cast<const T*>(a.dx) + e, n, f);
        if (a.d.limit != 0) drop8(a.d, step, a.d.first + e, f);
        add8(acc, f);
    }
    store_unit(static_cast<G*>(a.dp) + t * a.C + c, n, acc);
}

// [lo, hi) holds the first position whose key is at least v (hi: none before it); one step of the
// search by a wave leaves at most a 64th of it.
__device__ __forceinline__ void narrow(const unsigned* key, unsigned long v, int lane, int& lo, int& hi) {
    const int n = hi - lo;
    if (n <= 0) return;
    const int step = (n + 63) >> 6, at = lo + static_cast<int>(min(static_cast<long>(lane) * step + step - 1, n - 1L));
    const unsigned long less = __ballot(key[at] < v);  // (a run of ones from lane 0 on)
    const int k = __popcll(less);
    const int end = lo + static_cast<int>(min(static_cast<long>(k) * step + step - 1, n - 1L));  // key[end] >= v, if any
    if (k == 64) { lo = hi; return; }
    lo = lo + static_cast<int>(min(static_cast<long>(k) * step, static_cast<long>(n)));
    hi = end;
}

template <class G>
__device__ __forceinline__ void zero_absent(const BwdArgs& a, long block) {
    const int lane = threadIdx.x & 63;
    const long v = block * 64 + lane;
    // The first position whose key is at least v: the wave looks at 64 places at a time for the first
    // and the last of its rows, then every lane between these (a memory round trip per step: 2 + 3
    // instead of 12 of them for 4000 tokens over 32000 rows).
    int lo = 0, hi = a.R;
    const unsigned long from = static_cast<unsigned long>(block) * 64;
    int lo1 = 0, hi1 = a.R;  // of the row behind the last one
    while (hi - lo > 0 || hi1 - lo1 > 0) {
        narrow(a.key, from, lane, lo, hi);
        narrow(a.key, from + 64, lane, lo1, hi1);
    }
    hi = lo1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.key[mid] < static_cast<unsigned long>(v)) lo = mid + 1; else hi = mid;
    }
    const unsigned long absent = __ballot(v < a.V && !(lo < a.R && a.key[lo] == static_cast<unsigned long>(v)));
    // the 64 rows are one stretch of memory, walked in (aligned) units of eight whatever the row length
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const unsigned C = static_cast<unsigned>(a.C), n = static_cast<unsigned>(min(64L, a.V - block * 64)) * C;
    G* rows = static_cast<G*>(a.dw) + block * 64 * a.C;
    for (unsigned e = threadIdx.x * 8; e < n; e += 2048) {
        const unsigned r = e / C, end = min(e + 8, n);
        if (end <= (r + 1) * C) {
            if ((absent >> r) & 1) store_unit(rows + e, static_cast<int>(end - e), zero);
        } else {  // the unit spans rows
            for (unsigned i = e; i < end; ++i)
                if ((absent >> (i / C)) & 1) rows[i] = static_cast<G>(0.f);
        }
    }
}

template <class T, class G>
__global__ void __launch_bounds__(256) embedding_bwd_kernel(BwdArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned block = blockIdx.x;
    if (block < a.sum_blocks) sum_chunk<T, G>(a, block * 4L + wave, lane);
    else if (block < a.sum_blocks + a.pos_blocks) sum_position<T, G>(a, (block - a.sum_blocks) * 4L + wave, lane);
    else zero_absent<G>(a, block - a.sum_blocks - a.pos_blocks);
}

// One workgroup per chunk and 512 columns: where a run begins in the chunk and goes on, its waves
// sum the parts of the chunks behind, every eighth each, and the first adds them up.
template <class G>
__global__ void __launch_bounds__(512) embedding_join_kernel(BwdArgs a) {
    __shared__ float part[8][512];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ch = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs;
    const int p0 = ch * a.chunk, pe = p0 + a.chunk;  // (the last chunk has no join)
    if (pe >= a.R) return;
    // the keys at the chunk's borders and at the starts of those behind it, read together
    const int at = lane == 0 ? p0 - 1 : lane == 1 ? p0 : lane == 2 ? pe - 1 : pe;
    const unsigned edge = a.key[max(at, 0)];
    auto start = [&](int c) { return c < a.chunks ? a.key[static_cast<long>(c) * a.chunk] : 0xFFFFFFFFu; };
    unsigned first = start(ch + 1 + lane);
    const unsigned k = __builtin_amdgcn_readlane(edge, 3);
    if (__builtin_amdgcn_readlane(edge, 2) != k || k >= static_cast<unsigned>(a.V)) return;
    if (p0 > 0 && __builtin_amdgcn_readlane(edge, 1) == k && __builtin_amdgcn_readlane(edge, 0) == k)
        return;  // it began before the chunk
    // chunks behind this one whose first key is k hold a part in head[]
    int more = 0;
    for (int c0 = ch + 1;; c0 += 64) {
        if (c0 > ch + 1) first = start(c0 + lane);
        const unsigned long same = __ballot(first == k);
        more += __popcll(same);
        if (same != ~0UL) break;
    }
    const long c = slab * 512L + lane * 8;
    const int n = a.C - c >= 8 ? 8 : static_cast<int>(a.C - c);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n > 0) {
#pragma unroll 4
        for (int m = wave; m < more; m += 8) {
            float f[8];
            load_unit(a.head + static_cast<long>(ch + 1 + m) * a.C + c, n, f);
            add8(acc, f);
        }
    }
    store8(&part[wave][lane * 8], acc);
    __syncthreads();
    if (wave != 0 || n <= 0) return;
    load_unit(a.tail + static_cast<long>(ch) * a.C + c, n, acc);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        float f[8];
        load8(&part[w][lane * 8], f);
        add8(acc, f);
    }
    write_row<G>(a, k, c, n, acc);
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

// positions per chunk: enough chunks to fill the chip, up to 32 rows per wave; up to eight rows (two
// batches) are one chunk, which spares the launch of the join (8 tokens of 50257 x 768: 18.4 -> 16.5 us;
// 16 tokens as one chunk: 13.8 -> 19.2 of 20316 x 150)
int chunk_of(long R, int slabs) {
    int chunk = kMaxChunk;
    if (R <= 8) return chunk;
    while (chunk > 4 && R * slabs / chunk < 2048) chunk >>= 1;
    return chunk;
}

template <class T, class G>
int bwd(BwdArgs a, hipStream_t s) {
    const long sum = (static_cast<long>(a.chunks) * a.slabs + 3) / 4;
    const long pos = a.dp != nullptr ? (a.T * a.slabs + 3) / 4 : 0;
    const long zero = a.accumulate ? 0 : (a.V + 63) / 64;
    if (sum + pos + zero > kMaxBlocks) return -3;
    a.sum_blocks = static_cast<unsigned>(sum);
    a.pos_blocks = static_cast<unsigned>(pos);
    hipLaunchKernelGGL((embedding_bwd_kernel<T, G>), dim3(static_cast<unsigned>(sum + pos + zero)), dim3(256),
                       0, s, a);
    if (a.chunks > 1)
        hipLaunchKernelGGL((embedding_join_kernel<G>), dim3(static_cast<unsigned>(a.chunks) * a.slabs), dim3(512),
                           0, s, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace

extern "C" {

// The arguments of a call as one block.
// Forward: table [V][C]; pos (may be null): [>= T][C]; out [B][T][C]; type: 0 float, 1 bf16, 2 half
// (of all three).
// Backward: key / order: from nf_token_order, or both null: made here from the tokens.  dx: B T rows
// of C.  dw [V][C]: written everywhere, or (accumulate) added to where tokens are.  dp (may be null):
// rows 0 .. T - 1 are written.  type: of dx; grad_type: of dw and dp (0, or the type of dx).
struct EmbeddingArgs {
    const long* tokens;
    union { const void* table; const void* dx; };
    union { const void* pos; void* dp; };
    union { void* out; void* dw; };
    const unsigned *key, *order;
    float* scratch;
    const long* step_at;
    long padding, B, T, V, C, first;
    unsigned long long seed;
    double scale;
    unsigned limit, step;
    int type, grad_type, accumulate, unused;
};

int nf_embedding_args_size() { return static_cast<int>(sizeof(EmbeddingArgs)); }

int nf_embedding_fwd(const EmbeddingArgs* args, hipStream_t s) {
    const EmbeddingArgs& a = *args;
    if (a.B <= 0 || a.T <= 0 || a.V <= 0 || a.C <= 0 || a.limit > 65535u || a.first < 0) return -1;
    const DropRows d = drop_rows(a.limit, a.seed, a.step_at, a.step, a.first);
    const float scale = static_cast<float>(a.scale);
    switch (a.type) {
    case 0: return fwd<float>(a.tokens, a.table, a.pos, a.out, a.B * a.T, a.T, a.V, a.C, scale, d, s);
    case 1: return fwd<bf16>(a.tokens, a.table, a.pos, a.out, a.B * a.T, a.T, a.V, a.C, scale, d, s);
    case 2: return fwd<half>(a.tokens, a.table, a.pos, a.out, a.B * a.T, a.T, a.V, a.C, scale, d, s);
    default: return -1;
    }
}

// unsigned words of scratch that nf_token_order needs
long nf_token_order_words(long R) {
    return R <= kRankRows ? 0 : 2 * R + kMaxPasses * kMaxTiles * kDigits;
}

// key[i]: the i-th smallest token (V: none, or the padding token), order[i]: its row; equal
// tokens in the order of their rows.
int nf_token_order(const long* tokens, unsigned* key, unsigned* order, unsigned* scratch, long R, long V,
                   long padding, hipStream_t s) {
    if (R <= 0 || R >= (1L << 31) || V <= 0 || V >= (1L << 31)) return -1;
    const unsigned v = static_cast<unsigned>(V);
    if (R <= kRankRows) {
        hipLaunchKernelGGL(rank_kernel, dim3(static_cast<unsigned>((R + 15) / 16)), dim3(64 * kRankWaves), 0, s,
                           tokens, v, padding, key, order, static_cast<int>(R));
        return static_cast<int>(hipGetLastError());
    }
    const int rounds = static_cast<int>((R + kMaxTiles * 256L - 1) / (kMaxTiles * 256L));
    const dim3 grid(static_cast<unsigned>((R + rounds * 256L - 1) / (rounds * 256L)));
    unsigned *other_key = scratch, *other_order = scratch + R, *count = scratch + 2 * R;
    int passes = 1;
    while (passes < kMaxPasses && (v >> (8 * passes)) != 0) ++passes;
    const unsigned *from = nullptr, *from_order = nullptr;
    hipLaunchKernelGGL(digit_count_kernel, grid, dim3(256), 0, s, tokens, v, padding, count, R, rounds, passes - 1);
    for (int p = 0; p < passes; ++p) {
        const bool last = (passes - p) & 1;  // the passes alternate, the last one ends in key / order
        unsigned *to = last ? key : other_key, *to_order = last ? order : other_order;
        const long* tok = p == 0 ? tokens : nullptr;
        unsigned* now = count + p * kMaxTiles * kDigits;
        hipLaunchKernelGGL(digit_move_kernel, grid, dim3(256), 0, s, tok, from, from_order, v, padding, now,
                           p + 1 < passes ? now + kMaxTiles * kDigits : nullptr, to, to_order, R, rounds, 8 * p);
        from = to;
        from_order = to_order;
    }
    return static_cast<int>(hipGetLastError());
}

// 32-bit words of scratch that nf_embedding_bwd needs (`ordered`: with key and order given)
long nf_embedding_bwd_words(long R, long C, int ordered) {
    const int chunk = chunk_of(R, static_cast<int>((C + 511) / 512));
    return 2 * ((R + chunk - 1) / chunk) * C + (ordered ? 0 : 2 * R + nf_token_order_words(R));
}

int nf_embedding_bwd(const EmbeddingArgs* args, hipStream_t s) {
    const EmbeddingArgs& in = *args;
    const long B = in.B, T = in.T, V = in.V, C = in.C;
    if (B <= 0 || T <= 0 || V <= 0 || C <= 0 || in.limit > 65535u || in.first < 0) return -1;
    if (V >= (1L << 31) || C >= (1L << 25) || B >= (1L << 31) || T >= (1L << 31) || B * T >= (1L << 31)) return -3;
    if (in.grad_type != 0 && in.grad_type != in.type) return -1;
    BwdArgs a = {};
    a.dx = in.dx; a.dw = in.dw; a.dp = in.dp;
    a.B = B; a.T = T; a.V = V; a.C = C;
    a.R = static_cast<int>(B * T);
    a.slabs = static_cast<int>((C + 511) / 512);
    a.chunk = chunk_of(a.R, a.slabs);
    a.chunks = static_cast<int>((a.R + static_cast<long>(a.chunk) - 1) / a.chunk);
    a.head = in.scratch;
    a.tail = in.scratch + static_cast<long>(a.chunks) * C;
    a.accumulate = in.accumulate;
    a.scale = static_cast<float>(in.scale);
    a.d = drop_rows(in.limit, in.seed, in.step_at, in.step, in.first);
    if (static_cast<long>(a.chunks) * a.slabs > (1L << 22)) return -3;
    a.key = in.key;
    a.order = in.order;
    if (a.key == nullptr || a.order == nullptr) {
        unsigned* words = reinterpret_cast<unsigned*>(in.scratch + 2 * static_cast<long>(a.chunks) * C);
        const int status = nf_token_order(in.tokens, words, words + a.R, words + 2L * a.R, a.R, V, in.padding, s);
        if (status != 0) return status;
        a.key = words;
        a.order = words + a.R;
    }
    switch (in.type * 4 + in.grad_type) {
    case 0: return bwd<float, float>(a, s);
    case 4: return bwd<bf16, float>(a, s);
    case 5: return bwd<bf16, bf16>(a, s);
    case 8: return bwd<half, float>(a, s);
    case 10: return bwd<half, half>(a, s);
    default: return -1;
    }
}

}  // extern "C"
