// Causal attention with grouped heads over packed sequences whose keys and values are rows of a cache:
//
//   query i of a sequence (n queries, m keys) sees keys j <= m - n + i
//   out[i] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * (q_i . k_j) - top_i)         (nothing seen: zeros)
//
// in one pass over the keys with a running maximum and sum.  The rows of one key/value head are its group's heads of every
// query: row r of a sequence is query r / group, head r % group, so a key read serves the whole group.
//
// Scores are computed transposed, S^T = K Q^T, on the 32x32x16 matrix instruction: a lane then holds 16 keys of ONE row,
// the softmax statistics of a row are plain registers of its two lanes, and the exponentials, rounded to 16 bits, already
// lie as the second product O^T = V^T P^T wants them -- its contraction over keys may run in any order, and V's rows are
// read (transposed, from the LDS) in the order in which the lanes hold P.  P never leaves the registers.
//
// Two forms.  KEYS (single tokens: all rows of a tile fit one wavefront's 32): every wavefront takes its own tiles of 32 keys, and the
// keys may be split over workgroups.  TILE (prompts): the wavefronts of a workgroup take 32 rows each and share tiles of 64 keys;
// one workgroup per tile of 128 rows, or (few rows against many keys) workgroups with equal shares of all tiles' keys.
// Unnormalised sums and statistics of parts go to a workspace, and attention_join_kernel adds them up in their order.
//
// Rounding: products of 16-bit values summed in 32 bits; statistics, sums and rescaling in 32 bits; p is rounded to 16 bits
// for the second product (half a step of p each, bf16 2^-8 and fp16 2^-11 of it: the terms' errors average out) and for the sum of
// weights that divides it, the result once.
// The maximum is followed only where weights relative to the last one outgrow 2^15: most tiles look for none and rescale nothing.
#include <cmath>

#include "internal.hpp"
#include "lanes.hpp"

namespace sptmm {
namespace {

typedef unsigned short u16;
typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) unsigned short u16x4;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

struct AttnParams {
    const u16 *q, *k, *v;
    u16 *out;
    int64_t q_stride, k_stride, v_stride, out_stride, kv_rows;
    const int *q_start, *kv_start, *kv_len;
    int batch, total_q, q_heads, kv_heads, group, dim;
    float c;        // scale * log2(e)
    int slots;      // row tiles, over all sequences (an upper bound)
    int splits, chunk;  // KEYS: of every sequence's keys
    int log_rows;       // of a tile of the shares
    int shares;         // TILE: workgroups that take equal shares of all tiles' blocks of keys; 0: one workgroup per tile
    float *part_o;    // unnormalised sums: KEYS [split][query * q_heads + head][dim], TILE [share][0, 1][row of the tile][dim]
    float2 *part_ml;  // likewise: the maximum that the sums are relative to (of raw scores), sum
};

template <int T> __device__ __forceinline__ f32x16 mfma(u16x8 a, u16x8 b, f32x16 c)
{
    if constexpr (T == SPTMM_X_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int T> __device__ __forceinline__ u16 narrow(float x)
{
    if constexpr (T == SPTMM_X_F16) return __builtin_bit_cast(u16, (_Float16)x);
    return __builtin_bit_cast(u16, (__bf16)x);
}
// the two values of a word added to a 32-bit sum
template <int T> __device__ __forceinline__ float add_two(unsigned x, float sum)
{
    typedef __attribute__((ext_vector_type(2))) _Float16 h2;
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
    if constexpr (T == SPTMM_X_F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{(_Float16)1.f, (_Float16)1.f}, sum, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, x), b2{(__bf16)1.f, (__bf16)1.f}, sum, false);
}
// a lane's value and that of the lane 32 further (mod 64)
struct Halves {
    float a, b;
};
__device__ __forceinline__ Halves halves(float x)
{
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];  // (a bit cast of a vector's element itself reads its first element)
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ float halves_max(float x)
{
    const Halves h = halves(x);
    return fmaxf(h.a, h.b);
}
__device__ __forceinline__ float halves_sum(float x)
{
    const Halves h = halves(x);
    return h.a + h.b;
}

// One row tile of one sequence.  Tiles are found without a table: sequence b owns the slots from (first row of b) / TM + b
// on, which leaves it at least as many as it has tiles; what the arrays hold is clamped to the buffers' sizes, so that no
// content of theirs can send an access astray.
struct Tile {
    int q0, nq, k0, nk, row0, rows;  // first query, queries, first cache row, keys; first row of the tile, rows of the sequence
};

// A sequence's arrays, read by one lane and cut to the buffers
struct Seq {
    int q0, nq, k0, nk;
};
__device__ __forceinline__ Seq sequence(const AttnParams &p, int b)
{
    const int a = p.q_start[b], e = p.q_start[b + 1], at = p.kv_start ? p.kv_start[b] : a, len = p.kv_len ? p.kv_len[b] : e - a;
    Seq s;
    s.q0 = min(max(a, 0), p.total_q);
    s.nq = max(min(max(e, 0), p.total_q) - s.q0, 0);
    const bool there = at >= 0 && at < p.kv_rows;
    s.k0 = there ? at : 0;
    s.nk = there ? (int)min((int64_t)max(len, 0), p.kv_rows - at) : 0;
    return s;
}

template <int LOG_TM> __device__ __forceinline__ bool find_tile(const AttnParams &p, int slot, Tile *t)
{
    const int lane = threadIdx.x & 63;
    bool found = false;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const int b = b0 + lane;
        const Seq s = sequence(p, min(b, p.batch - 1));
        const int first = (int)(((int64_t)s.q0 * p.group) >> LOG_TM) + b;
        const int c = __popcll(__ballot(b < p.batch && first <= slot));
        if (c == 0) break;
        found = true;
        t->q0 = __builtin_amdgcn_readlane(s.q0, c - 1);
        t->nq = __builtin_amdgcn_readlane(s.nq, c - 1);
        t->k0 = __builtin_amdgcn_readlane(s.k0, c - 1);
        t->nk = __builtin_amdgcn_readlane(s.nk, c - 1);
        t->row0 = slot - __builtin_amdgcn_readlane(first, c - 1);
        if (c < 64) break;
    }
    if (!found || t->row0 > t->nq * p.group >> LOG_TM) return false;
    t->rows = t->nq * p.group;
    t->row0 <<= LOG_TM;
    return t->row0 >= 0 && t->row0 < t->rows;
}

// Tiles of 128 rows and their keys as one row of blocks of 128 keys, for the sharing of the work: sequence by sequence, in it head by
// head, tile by tile, all of a sequence's tiles with the blocks of all its keys (one at least, so that a tile without keys is
// written too).  Found, like the tiles, by every wavefront from the sequences' arrays alone.
constexpr int LOG_TILE = 7, TILE_ROWS = 1 << LOG_TILE, LOG_BLOCK = 7, LEAST_BLOCKS = 2 /* of a share */, MOST_SHARES = 512;

__device__ __forceinline__ int tiles_of(const AttnParams &p, const Seq &s) { return (s.nq * p.group + (1 << p.log_rows) - 1) >> p.log_rows; }
__device__ __forceinline__ int blocks_of(const Seq &s) { return max(1, (s.nk + (1 << LOG_BLOCK) - 1) >> LOG_BLOCK); }
// of sequence b (none: 0)
__device__ __forceinline__ int64_t seq_blocks(const AttnParams &p, int b, Seq *s)
{
    *s = sequence(p, min(b, p.batch - 1));
    return b < p.batch ? (int64_t)tiles_of(p, *s) * p.kv_heads * blocks_of(*s) : 0;
}
// a value that all lanes share, in scalar registers (the vector ones are the inner loop's)
__device__ __forceinline__ int64_t uniform(int64_t x) { return (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ int64_t wave_sum(int64_t x)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor((long long)x, o, 64);
    return uniform(x);
}
__device__ __forceinline__ int64_t all_blocks(const AttnParams &p)
{
    int64_t sum = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        Seq s;
        sum += seq_blocks(p, b0 + (threadIdx.x & 63), &s);
    }
    return wave_sum(sum);
}
__device__ __forceinline__ int64_t share(const AttnParams &p, int64_t all) { return max((all + p.shares - 1) / p.shares, (int64_t)LEAST_BLOCKS); }

// A place in the row of blocks: sequence, tile (of its heads' tiles, one head's after another), block
struct Place {
    int q0, nq, k0, nk, tiles, blocks, tile, block;
};
// the place `rest` blocks into the sequence that lane c holds
__device__ __forceinline__ Place place(const AttnParams &p, const Seq &s, int c, int64_t rest)
{
    Place a;
    a.q0 = __builtin_amdgcn_readlane(s.q0, c), a.nq = __builtin_amdgcn_readlane(s.nq, c);
    a.k0 = __builtin_amdgcn_readlane(s.k0, c), a.nk = __builtin_amdgcn_readlane(s.nk, c);
    a.tiles = __builtin_amdgcn_readlane(tiles_of(p, s), c), a.blocks = __builtin_amdgcn_readlane(blocks_of(s), c);
    a.tile = __builtin_amdgcn_readfirstlane((int)(rest / a.blocks));
    a.block = __builtin_amdgcn_readfirstlane((int)(rest - (int64_t)a.tile * a.blocks));
    return a;
}
// blocks of the sequences from b0 on up to and with this lane's
__device__ __forceinline__ int64_t scan_blocks(const AttnParams &p, int b0, Seq *s, int64_t *mine)
{
    const int lane = threadIdx.x & 63;
    int64_t upto = *mine = seq_blocks(p, b0 + lane, s);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up((long long)upto, o, 64);
        upto += lane >= o ? x : 0;
    }
    return upto;
}
__device__ __forceinline__ bool find_block(const AttnParams &p, int64_t u, Place *a)
{
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        Seq s;
        int64_t mine;
        const int64_t upto = scan_blocks(p, b0, &s, &mine);
        const int c = __popcll(__ballot(upto <= u));
        if (c < 64) {
            *a = place(p, s, c, u - uniform(__shfl((long long)(upto - mine), c, 64)));
            return true;
        }
        u -= uniform(__shfl((long long)upto, 63, 64));
    }
    return false;
}
// where share i begins, and how many blocks a share has
__device__ __forceinline__ bool find_share(const AttnParams &p, int i, Place *a, int64_t *per)
{
    if (p.batch > 64) {
        *per = uniform(share(p, all_blocks(p)));
        return find_block(p, i * *per, a);
    }
    Seq s;
    int64_t mine;
    const int64_t upto = scan_blocks(p, 0, &s, &mine), all = uniform(__shfl((long long)upto, 63, 64));
    *per = uniform(share(p, all));
    const int64_t u = i * *per;
    if (u >= all) return false;
    const int c = __popcll(__ballot(upto <= u));
    *a = place(p, s, c, u - uniform(__shfl((long long)(upto - mine), c, 64)));
    return true;
}

// ------------------------------------------------------------------------------------------------ tiles in the LDS
// A tile is KT rows of DP values in row order; the 16-byte pieces of a row are permuted among themselves by a function of
// the row so that the reads below meet different banks: K is read 16 bytes a lane, one piece of 32 rows at a time; V four
// values a lane, four pieces of eight rows at a time, transposed on the way.
template <int DP> __device__ __forceinline__ int swizzle_k(int row) { return DP == 64 ? (row >> 1) & 7 : row & 15; }
template <int DP> __device__ __forceinline__ int swizzle_v(int row) { return DP == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }

typedef __attribute__((address_space(3))) void *lds_ptr;

// Rows straight from memory into the LDS: one instruction of a wavefront moves 64 pieces (1 KiB).  Pieces behind the last
// row or behind the head's last element lie outside the buffer that the descriptor names and arrive as zeros.  STREAM: loads that
// do not stay in the caches.
template <int DP, int KT, int WAVES, bool STREAM = false> struct Loader {
    static constexpr int PIECES = DP / 8, PER = KT * PIECES / 64 / WAVES;
    static_assert(PER >= 1, "every wavefront loads something");
    int off[PER];
    __device__ __forceinline__ void init(int64_t stride, int dim, int lane, int wave, bool is_v)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = (i * WAVES + wave) * 64 + lane, row = at / PIECES;
            const int piece = (at % PIECES) ^ (is_v ? swizzle_v<DP>(row) : swizzle_k<DP>(row));
            off[i] = piece * 8 < dim ? (int)(row * stride * 2) + piece * 16 : 0x7ffffff0;
        }
    }
    __device__ __forceinline__ void issue(const u16 *base, int64_t stride, int dim, int rows_left, char *lds, int wave) const
    {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass does not know buffer descriptors, and would drop kernels that name them)
        const int bytes = rows_left <= 0 ? 0 : (int)((min(rows_left, KT) - 1) * stride * 2) + dim * 2;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(lds + (i * WAVES + wave) * 1024), 16, off[i], 0, 0, STREAM ? 2 : 0);
#endif
    }
};

// ------------------------------------------------------------------------------------------------ one wavefront's rows
template <int T, int DP, int KT> struct Rows {
    enum { CLEAN, EDGE };
    static constexpr int KS = DP / 16, DS = DP / 32, KB = KT / 32;
    u16x8 qf[KS];
    f32x16 o[DS];
    float top, sum;  // running maximum of the raw scores, and this lane's share of the sum
    int lim;         // last key this lane's row sees
    int k_at, v_at[DS];

    __device__ __forceinline__ void init(const AttnParams &p, const Tile &t, int kv_head, int row, bool valid, int lane)
    {
        const int half = lane >> 5;
        const int i = row / p.group, head = kv_head * p.group + row - i * p.group;
        lim = t.nk - t.nq + i;
        const u16 *q = p.q + (int64_t)(t.q0 + i) * p.q_stride + (int64_t)head * p.dim + 8 * half;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (valid && 16 * s + 8 * half < p.dim) qf[s] = *reinterpret_cast<const u16x8 *>(q + 16 * s);
        }
#pragma unroll
        for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
        top = -INFINITY, sum = 0.f;
        // where this lane reads K (row lane % 32 of a block of 32, piece 2 s + half) and V (row 4 half + (lane % 16) / 4 of every
        // eight, four values from d = 32 b + 16 (lane / 16 % 2) + 4 (lane % 4) on)
        k_at = (lane & 31) * DP * 2 + ((half ^ swizzle_k<DP>(lane & 31)) << 4);
        const int vr = 4 * half + ((lane & 15) >> 2);
#pragma unroll
        for (int d = 0; d < DS; ++d) v_at[d] = vr * DP * 2 + (((4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swizzle_v<DP>(vr)) << 4) + (lane & 1) * 8;
    }

    // A row's p is zero at keys it does not see, and zero times an infinity is not zero.  Where some row of this wavefront does not
    // see every key that the tile holds (those before `end`; lo: the smallest last key of the rows), a tile of V with a value
    // that is not finite is added key by key, to the rows that see the key.
    __device__ __forceinline__ bool polluted(const char *v, int j0, int end, int lo) const
    {
        if (min(j0 + KT, end) - 1 <= lo) return false;
        const int lane = threadIdx.x & 63;
        // the largest magnitude of all the values' bits, as integers: an exponent of ones is above every finite value's
        typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
        u16x2 most = {0, 0};
#pragma unroll
        for (int i = 0; i < KT * DP / 512; ++i) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(v + (i * 64 + lane) * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned x = w[j] & 0x7fff7fffu;
                most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x));
            }
        }
        constexpr unsigned short E = T == SPTMM_X_F16 ? 0x7c00 : 0x7f80;
        return __ballot(most[0] >= E || most[1] >= E) != 0;
    }

    // V for the 32 values of d from 32 b on: for step t the keys 16 t + 4 half + {0..3} and + 8, which are those of this lane's P
    __device__ __forceinline__ void v_frags(const char *v, int b, u16x8 (&f)[2 * KB]) const
    {
        typedef __attribute__((address_space(3))) s16x4 *lds4;
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t) {
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(v + v_at[b] + t * 16 * DP * 2));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(v + v_at[b] + (t * 16 + 8) * DP * 2));
            f[t] = __builtin_bit_cast(u16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }

    // One tile of keys, from j0 on.  CLEAN: every row of this wavefront sees all of it; EDGE: some do not.  bad: see `polluted`.
    template <int KIND> __device__ __forceinline__ void step(const AttnParams &p, const char *k, const char *v, int j0 = 0, int lo = 0, bool bad = false)
    {
        const int half = (threadIdx.x & 63) >> 5;
        f32x16 s[KB];
        auto score = [&] {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[b][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int b = 0; b < KB; ++b)
                    s[b] = mfma<T>(*reinterpret_cast<const u16x8 *>(k + (k_at ^ (ks << 5)) + b * 32 * DP * 2), qf[ks], s[b]);
            if (KIND == EDGE && j0 + KT - 1 > lo) {
                const int last = lim - j0 - 4 * half;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[b][e] = b * 32 + 8 * (e >> 2) + (e & 3) <= last ? s[b][e] : -INFINITY;
            }
        };
        u16x8 pf[2 * KB];
        // the weights relative to `top`, rounded into pf; their 32-bit sum, of the rounded values: a row of one key is then that key's value
        // exactly, and a few keys' roundings cancel.  fp16: p is held 2^7 larger, so that what rounds to zero is below 2^-32 of
        // the largest.
        auto weigh = [&] {
            const float at = (top == -INFINITY ? 0.f : top * p.c) - (T == SPTMM_X_F16 ? 7.f : 0.f);
            float part[4] = {0.f, 0.f, 0.f, 0.f};
            // Summed behind all exponentials, or (heads of 256, one wavefront per SIMD) each pair at once: 3000 tokens of 256 169 us and 110,
            // 8192 of 128 339 and 349.  (Sums of the weights before their rounding: 129 and 329, now 330, chunks 175 and 182.)
#pragma unroll
            for (int t = 0; t < 2 * KB; ++t) {
                auto weight = [&](int e) { return __builtin_amdgcn_exp2f(fmaf(s[t >> 1][8 * (t & 1) + e], p.c, -at)); };
                if constexpr (DP == 256) {
                    u32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = weight(2 * i), y = weight(2 * i + 1);
                        const unsigned two = narrow<T>(x) | (unsigned)narrow<T>(y) << 16;
                        w[i] = two;
                        part[i] = add_two<T>(two, part[i]);
                    }
                    pf[t] = __builtin_bit_cast(u16x8, w);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) pf[t][e] = narrow<T>(weight(e));
                }
            }
            if constexpr (DP != 256)
#pragma unroll
                for (int t = 0; t < 2 * KB; ++t) {
                    const u32x4 w = __builtin_bit_cast(u32x4, pf[t]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const unsigned two = w[i];
                        part[i & 1] = add_two<T>(two, part[i & 1]);
                    }
                }
            return (part[0] + part[1]) + (part[2] + part[3]);
        };
        score();
        float tile_sum = weigh();
        // Weights relative to an old maximum are as good as any while they fit: only where they outgrow 2^15 (or there is no maximum
        // yet) is the tile's maximum looked for and followed, and the tile weighed again.  An fp16 weight is then below 2^16 always.
        if (__ballot(tile_sum > 32768.f || top == -INFINITY)) {
            score();
            float mx = s[0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[b][e]);
            const float now = fmaxf(top, halves_max(mx)), f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((top - now) * p.c);
#pragma unroll
            for (int d = 0; d < DS; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= f;
            sum *= f;
            top = now;
            tile_sum = weigh();
        }
        sum += tile_sum;
        if (KIND == EDGE && bad) {
            const f32x16 zero = {0.f};
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                u16x8 vf[2 * KB];
                v_frags(v, d, vf);
#pragma unroll
                for (int t = 0; t < 2 * KB; ++t)
#pragma unroll 1
                    for (int x = 0; x < 16; ++x) {  // element x % 8 of the lower (x < 8) or the upper lanes' eight keys of step t
                        const int e = x & 7, key = j0 + 16 * t + (e < 4 ? e : e + 4) + 4 * (x >> 3);
                        u32x4 only;
#pragma unroll
                        for (int w = 0; w < 4; ++w) only[w] = half == x >> 3 && w == e >> 1 ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
                        const f32x16 n = mfma<T>(__builtin_bit_cast(u16x8, __builtin_bit_cast(u32x4, vf[t]) & only), __builtin_bit_cast(u16x8, __builtin_bit_cast(u32x4, pf[t]) & only), zero);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] += key <= lim ? n[i] : 0.f;
                    }
            }
        } else {
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                u16x8 vf[2 * KB];
                v_frags(v, d, vf);
#pragma unroll
                for (int t = 0; t < 2 * KB; ++t) o[d] = mfma<T>(vf[t], pf[t], o[d]);
            }
        }
    }
};

// this wavefront's loads into the LDS have landed and its reads are done, and so for the whole workgroup
__device__ __forceinline__ void lds_arrived() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int T> __device__ __forceinline__ void write4(const AttnParams &p, const Tile &t, int kv_head, int row, int d, f32x4 x)
{
    const int i = row / p.group, head = kv_head * p.group + row - i * p.group;
    u16x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = narrow<T>(x[e]);
    *reinterpret_cast<u16x4 *>(p.out + (int64_t)(t.q0 + i) * p.out_stride + (int64_t)head * p.dim + d) = y;
}

// ------------------------------------------------------------------------------------------------ TILE: rows over wavefronts
// Bound by the matrix units' feed: one prompt of 8192 tokens, 20 heads of 128 on 5, bf16: 344 GFLOP in 315 to 347 us by card, 1.0 to 1.1 PFLOP/s, where
// a product of two 8192 x 8192 matrices reaches 1.21; matrix units busy 54 % of the cycles, at 1.7 to 1.8 GHz.  64 KB of LDS leave two workgroups to a compute unit, and
// one's exponentials run beside the other's products; of the time, the exponentials alone are a tenth, the loads 3 %.  Four
// wavefronts of 32 rows share each tile of K and V through the LDS (without bank conflicts); of 256 rows: slower, one workgroup a unit.
//
// Keys begin .. end - 1 (begin a multiple of the tile of keys, end one too or the last key that a row sees) for the 32 * WAVES rows of t.
// part < 0: the rows are done and written; else their sums become part `part` in the workspace.
template <int T, int DP, int KT, int WAVES> __device__ __forceinline__ void tile_rows(const AttnParams &p, const Tile &t, int kv_head, int begin, int end, int i_last, char *k_a, char *k_b,
                                                                                      char *v_a, char *v_b, int part)
{
    unsigned thread = threadIdx.x;
    asm volatile("" : "+v"(thread));  // (what follows from it is computed here and not kept in registers from one call to the next)
    const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    Loader<DP, KT, WAVES> lk, lv;
    lk.init(p.k_stride, p.dim, lane, wave, false);
    lv.init(p.v_stride, p.dim, lane, wave, true);
    const u16 *k = p.k + (int64_t)t.k0 * p.k_stride + (int64_t)kv_head * p.dim, *v = p.v + (int64_t)t.k0 * p.v_stride + (int64_t)kv_head * p.dim;

    const int n = begin < end ? (end - begin + KT - 1) / KT : 0;
    // tiles that every row of the workgroup sees whole, in pairs: the two pairs of buffers alternate by name, so that the compiler
    // knows which loads a read has to wait for
    const int clean = max(0, min(t.nk - t.nq + t.row0 / p.group + 1, end) - begin) / KT & ~1;
    auto load = [&](int i, char *kl, char *vl) {  // behind the last tile: zeros, without an access to memory
        const int j = begin + i * KT;
        lk.issue(k + (int64_t)j * p.k_stride, p.k_stride, p.dim, end - j, kl, wave);
        lv.issue(v + (int64_t)j * p.v_stride, p.v_stride, p.dim, end - j, vl, wave);
    };
    load(0, k_a, v_a);
    typedef Rows<T, DP, KT> R;
    R r;
    const int row = t.row0 + wave * 32 + (lane & 31);
    const bool valid = row < t.rows;
    r.init(p, t, kv_head, valid ? row : t.rows - 1, valid, lane);
    const int row_w = t.row0 + wave * 32, lo = t.nk - t.nq + row_w / p.group;
    const int hi = row_w < t.rows ? t.nk - t.nq + min(i_last, (row_w + 31) / p.group) : -1;
    int i = 0;
    for (; i < clean; i += 2) {
        lds_arrived();
        load(i + 1, k_b, v_b);
        r.template step<R::CLEAN>(p, k_a, v_a);
        lds_arrived();
        load(i + 2, k_a, v_a);
        r.template step<R::CLEAN>(p, k_b, v_b);
    }
    for (; i < n; ++i) {
        int j = begin + i * KT;
        lds_arrived();
        load(i + 1, k_b, v_b);
        if (j <= hi) r.template step<R::EDGE>(p, k_a, v_a, j, lo, r.polluted(v_a, j, end, lo));
        if (++i >= n) break;
        j += KT;
        lds_arrived();
        load(i + 1, k_a, v_a);
        if (j <= hi) r.template step<R::EDGE>(p, k_b, v_b, j, lo, r.polluted(v_b, j, end, lo));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (nothing is on its way into the LDS when the workgroup gives it up)
    const float sum = halves_sum(r.sum), f = part < 0 ? 1.f / sum : 1.f;
    if (!valid) return;
    const bool none = r.lim < 0;
    const int64_t part_row = (int64_t)part * (32 * WAVES) + row - t.row0;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = 32 * d + 8 * e + 4 * (lane >> 5);
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = none ? 0.f : r.o[d][4 * e + i] * f;
            if (at >= p.dim) continue;
            if (part < 0) write4<T>(p, t, kv_head, row, at, x);
            else *reinterpret_cast<f32x4 *>(p.part_o + part_row * p.dim + at) = x;
        }
    if (part >= 0 && lane < 32) p.part_ml[part_row] = float2{r.top, sum};
}

// SHARED: the blocks of keys of all tiles, tile after tile, are cut into equal shares, one a workgroup; a share may end within a tile
// and go on in the next.  A tile that lies in one share is written; others leave their sums, a workgroup at most two: of a
// tile that it ends (part 0) and of one that it begins (part 1).  Neighbouring shares, which read the same keys, go to one XCD.
// Four chunks of 130 to 250 tokens against 12000 to 20000 keys, 134 GFLOP: 160 us, and 17 for the join.
template <int T, int DP, int KT, int WAVES, bool SHARED> __global__ void __launch_bounds__(64 * WAVES, DP == 256 ? 1 : 2) attention_tile_kernel(const AttnParams p)
{
    __shared__ __attribute__((aligned(1024))) char k_a[KT * DP * 2], k_b[KT * DP * 2], v_a[KT * DP * 2], v_b[KT * DP * 2];
    Tile t;
    if constexpr (SHARED) {
        const int i = (int)(blockIdx.x % 8 * (p.shares / 8) + blockIdx.x / 8);
        Place a;
        int64_t per;
        if (!find_share(p, i, &a, &per)) return;
        for (int64_t left = per;;) {
            const int kv_head = a.tile / a.tiles, n = (int)min((int64_t)(a.blocks - a.block), left);
            t = {a.q0, a.nq, a.k0, a.nk, (a.tile - kv_head * a.tiles) << p.log_rows, a.nq * p.group};
            const int i_last = (min(t.row0 + 32 * WAVES, t.rows) - 1) / p.group, all = max(0, min(t.nk, t.nk - t.nq + i_last + 1));
            tile_rows<T, DP, KT, WAVES>(p, t, kv_head, min(a.block << LOG_BLOCK, all), min((a.block + n) << LOG_BLOCK, all), i_last, k_a, k_b, v_a, v_b, n == a.blocks ? -1 : 2 * i + (a.block == 0));
            if ((left -= n) == 0) return;
            a.block = 0;
            if (++a.tile == a.tiles * p.kv_heads && !find_block(p, (i + 1) * per - left, &a)) return;
            __syncthreads();  // (all are done with the tiles of keys)
        }
    } else {
        // A sequence's last rows, which see the most keys, first, and of all heads before the next rows: workgroups dispatched late
        // are short.  (All sequences' tiles in one order of the keys they see: eight chunks of up to 400 tokens 361 us, so 371; thirty
        // prompts of 30 to 1500 tokens 170, so 150.  Heads kept to their XCDs' L2s: one prompt of 8192, 5 heads, 341 and 346; 32 heads 524 and 510.)
        const int kv_head = (int)(blockIdx.x % (unsigned)p.kv_heads), slot = p.slots - 1 - (int)(blockIdx.x / (unsigned)p.kv_heads);
        if (!find_tile<LOG_TILE>(p, slot, &t)) return;
        const int i_last = (min(t.row0 + TILE_ROWS, t.rows) - 1) / p.group, all = min(t.nk, t.nk - t.nq + i_last + 1);
        tile_rows<T, DP, KT, WAVES>(p, t, kv_head, 0, all, i_last, k_a, k_b, v_a, v_b, -1);
    }
}

// ------------------------------------------------------------------------------------------------ KEYS: keys over wavefronts
// Bound by the cache's read: 32 sequences of 2000 to 8000 keys, 661 MB, 5.5 TB/s.  Nothing is shared between wavefronts but the
// sums at the end, so that each waits for its own loads only.  Two to a workgroup, as 128 KB of LDS for four leave one workgroup
// to a compute unit: 20 heads of 128 on 5, one token against 8000 keys 13.7 us and 18.6, 32 against 1500 36 and 40, 64: 55 and 54.
// Heads over 128 are far from this: the 32 offsets of a tile's loads do not fit the registers beside Q and O, every load waits for its
// own from scratch memory, and 16 heads of 256 on 4, 32 caches of 0 to 16384 keys, 1059 MB, take 1950 us (0.54 TB/s).
template <int T, int DP, int WAVES, bool STREAM> __global__ void __launch_bounds__(64 * WAVES, DP == 256 ? 1 : 2) attention_keys_kernel(const AttnParams p)
{
    constexpr int KT = 32, LOG_TM = 5, ONE = KT * DP * 2;
    __shared__ __attribute__((aligned(1024))) char k_a[WAVES * ONE], k_b[WAVES * ONE], v_a[WAVES * ONE], v_b[WAVES * ONE];
    __shared__ float tops[WAVES][32], sums[WAVES][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    if (!find_tile<LOG_TM>(p, (int)blockIdx.x, &t)) return;
    const int kv_head = blockIdx.y, split = blockIdx.z;
    const int rows = min(32, t.rows - t.row0), i_last = (t.row0 + rows - 1) / p.group, all = min(t.nk, t.nk - t.nq + i_last + 1);
    const int begin = split * p.chunk, end = split == p.splits - 1 ? all : min(all, begin + p.chunk);
    if (split && begin >= end) return;

    Loader<DP, KT, 1, STREAM> lk, lv;
    lk.init(p.k_stride, p.dim, lane, 0, false);
    lv.init(p.v_stride, p.dim, lane, 0, true);
    const u16 *k = p.k + (int64_t)t.k0 * p.k_stride + (int64_t)kv_head * p.dim, *v = p.v + (int64_t)t.k0 * p.v_stride + (int64_t)kv_head * p.dim;
    // this wavefront's tiles: every WAVES-th, one in use while the next is on its way
    constexpr int STRIDE = WAVES * KT;
    const int j0 = begin + wave * KT, n = j0 < end ? (end - j0 + STRIDE - 1) / STRIDE : 0;
    const int lo = t.nk - t.nq + t.row0 / p.group, whole = min(lo + 1, end) - j0, clean = (whole < KT ? 0 : (whole - KT) / STRIDE + 1) & ~1;
    auto load = [&](int i, char *kl, char *vl) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the tile that this load overwrites are done
        if (i < n) {
            const int j = j0 + i * STRIDE;
            lk.issue(k + (int64_t)j * p.k_stride, p.k_stride, p.dim, end - j, kl + wave * ONE, 0);
            lv.issue(v + (int64_t)j * p.v_stride, p.v_stride, p.dim, end - j, vl + wave * ONE, 0);
            if (i) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * Loader<DP, KT, 1, STREAM>::PER) : "memory");  // the tile before this one has landed
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    };
    typedef Rows<T, DP, KT> R;
    char *const ka = k_a + wave * ONE, *const kb = k_b + wave * ONE, *const va = v_a + wave * ONE, *const vb = v_b + wave * ONE;
    load(0, k_a, v_a);
    R r;
    const bool valid = (lane & 31) < rows;
    r.init(p, t, kv_head, t.row0 + (valid ? lane & 31 : 0), valid, lane);
    int i = 0;
    for (; i < clean; i += 2) {
        load(i + 1, k_b, v_b);
        r.template step<R::CLEAN>(p, ka, va);
        load(i + 2, k_a, v_a);
        r.template step<R::CLEAN>(p, kb, vb);
    }
    for (; i < n; ++i) {
        int j = j0 + i * STRIDE;
        load(i + 1, k_b, v_b);
        r.template step<R::EDGE>(p, ka, va, j, lo, r.polluted(va, j, end, lo));
        if (++i >= n) break;
        j += STRIDE;
        load(i + 1, k_a, v_a);
        r.template step<R::EDGE>(p, kb, vb, j, lo, r.polluted(vb, j, end, lo));
    }
    // the wavefronts' sums, brought to one maximum and added in wavefront order; a wavefront's part lies where its tiles lay.  Where a
    // wavefront has no maximum its sums are zeros, or NaN (the maximum passes over scores that are NaN), and are added as they are.
    const float sum = halves_sum(r.sum);
    if (lane < 32) tops[wave][lane] = r.top, sums[wave][lane] = sum;
    __syncthreads();
    float top = tops[0][lane & 31];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, tops[w][lane & 31]);
    const float f = r.top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((r.top - top) * p.c);
    constexpr int PER = ONE / 4096;  // blocks of 32 values of d that one array has room for
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = r.o[d][4 * e + i] * f;
            *reinterpret_cast<f32x4 *>((d < PER ? k_a : v_a) + wave * ONE + (d % PER) * 4096 + e * 1024 + lane * 16) = x;
        }
    __syncthreads();
    const int quads = p.dim / 4;
    for (int at = threadIdx.x; at < rows * quads; at += 64 * WAVES) {
        const int rr = at / quads, d4 = at - rr * quads, d = d4 >> 3, e = (d4 & 7) >> 1, from = (d4 & 1) * 32 + rr;
        const char *src = (d < PER ? k_a : v_a) + (d % PER) * 4096 + e * 1024 + from * 16;
        f32x4 x = *reinterpret_cast<const f32x4 *>(src);
        float best = tops[0][rr];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            x += *reinterpret_cast<const f32x4 *>(src + w * ONE);
            best = fmaxf(best, tops[w][rr]);
        }
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) total += sums[w][rr] * (tops[w][rr] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((tops[w][rr] - best) * p.c));
        const int row = t.row0 + rr, i = row / p.group;
        if (p.splits > 1) {
            const int64_t part_row = (int64_t)split * p.total_q * p.q_heads + (int64_t)(t.q0 + i) * p.q_heads + kv_head * p.group + row - i * p.group;
            if (d4 == 0) p.part_ml[part_row] = float2{best, total};
            *reinterpret_cast<f32x4 *>(p.part_o + part_row * p.dim + 4 * d4) = x;
        } else {
            const float inv = 1.f / total;
            const bool none = t.nk - t.nq + i < 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = none ? 0.f : x[c] * inv;
            write4<T>(p, t, kv_head, row, 4 * d4, x);
        }
    }
}

// ------------------------------------------------------------------------------------------------ parts joined
// One row's n parts, added in their order by WAVES wavefronts and written: the four of a workgroup where there are many parts
// (one token of 20 heads against 8000 keys, 63 parts: the call 13.6 us, by single wavefronts 16.8), one where there are few
// and many rows.  at(i): where part i lies.
template <int T, int WAVES, int MOST, typename At> __device__ __forceinline__ void join_row(const AttnParams &p, f32x4 (&parts)[4][64], int wave, int n, bool none, At at, u16 *out)
{
    constexpr int PER = MOST / 64;
    const int lane = threadIdx.x & 63;
    // every lane holds the weight of one part (and of those 64, 128, ... further)
    float2 ml[PER];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        ml[i] = lane + 64 * i < n ? p.part_ml[at(lane + 64 * i)] : float2{-INFINITY, 0.f};
        top = fmaxf(top, ml[i].x);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    float w[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        w[i] = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[i].x - top) * p.c);
        sum = fmaf(ml[i].y, w[i], sum);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    // four values a lane, and as many parts side by side as lanes are left, and every WAVES-th such group a wavefront's
    const int quads = p.dim / 4, log_l = quads <= 2 ? 1 : 32 - __builtin_clz(quads - 1), sub = lane >> log_l, d4 = lane & ((1 << log_l) - 1), step = 64 >> log_l;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int end = min(64, n - 64 * i);
        for (int s0 = wave * step; s0 < end; s0 += 4 * WAVES * step) {
            f32x4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)  // (four loads in flight; behind the last part: its values, left out below)
                x[u] = *reinterpret_cast<const f32x4 *>(p.part_o + at(min(64 * i + s0 + u * WAVES * step + sub, n - 1)) * p.dim + 4 * min(d4, quads - 1));
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int s = s0 + u * WAVES * step + sub;
                const float f = __shfl(w[i], s & 63, 64);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = s < end ? fmaf(x[u][e], f, o[e]) : o[e];
            }
        }
    }
    for (int l = 1 << log_l; l < 64; l <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], l, 64);
    if constexpr (WAVES == 4) {
        parts[wave][lane] = o;
        __syncthreads();
        o = (parts[0][lane] + parts[1][lane]) + (parts[2][lane] + parts[3][lane]);
    }
    if (wave || sub || d4 >= quads) return;
    const float inv = 1.f / sum;
    u16x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = narrow<T>(none ? 0.f : o[e] * inv);
    *reinterpret_cast<u16x4 *>(out + 4 * d4) = y;
}

// Per (query, head).  SHARED: the parts that the shares left of the row's tile, if they cut it; else the splits that hold keys the row sees.
template <int T, int WAVES, bool SHARED> __global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p)
{
    __shared__ __attribute__((aligned(16))) f32x4 parts[4][64];
    const int lane = threadIdx.x & 63, in_block = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = WAVES == 1 ? 0 : in_block;
    const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + in_block : blockIdx.x, all = (int64_t)p.total_q * p.q_heads;
    if (row >= all) return;
    const int query = (int)(row / p.q_heads), head = (int)(row - (int64_t)query * p.q_heads);
    // the sequence of this query: the last one that starts at or before it; the blocks before it, and all
    Seq s = {0, 0, 0, 0};
    int64_t before = 0, blocks = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const int b = b0 + lane;
        Seq mine;
        int64_t w = 0;
        if constexpr (SHARED) w = seq_blocks(p, b, &mine);
        else mine = sequence(p, min(b, p.batch - 1));
        const int c = __popcll(__ballot(b < p.batch && mine.q0 <= query));
        if (c) {
            s = {__builtin_amdgcn_readlane(mine.q0, c - 1), __builtin_amdgcn_readlane(mine.nq, c - 1), 0, __builtin_amdgcn_readlane(mine.nk, c - 1)};
            before = blocks + (lane < c - 1 ? w : 0);
        }
        blocks += w;
        if (!SHARED && c < 64) break;
    }
    // a row behind the last sequence; or starts that are out of order, whose count names a sequence behind the row: no part is its own
    if (query < s.q0 || query >= s.q0 + s.nq) return;
    u16 *const out = p.out + (int64_t)query * p.out_stride + (int64_t)head * p.dim;
    const int seen = s.nk - s.nq + (query - s.q0) + 1;
    if constexpr (SHARED) {
        const int64_t per = share(p, wave_sum(blocks));
        const int kv_head = head / p.group, r = (query - s.q0) * p.group + head - kv_head * p.group, mine = blocks_of(s);
        const int64_t first = wave_sum(before) + ((int64_t)kv_head * tiles_of(p, s) + (r >> p.log_rows)) * mine;
        const int i0 = (int)min(first / per, (int64_t)p.shares - 1), i1 = (int)min((first + mine - 1) / per, (int64_t)p.shares - 1);
        if (i0 == i1) return;  // written already
        join_row<T, WAVES, MOST_SHARES>(p, parts, wave, i1 - i0 + 1, seen <= 0, [&](int i) { return ((int64_t)(2 * (i0 + i) + (i == 0)) << p.log_rows) + (r & ((1 << p.log_rows) - 1)); }, out);
    } else {
        const int n = seen <= 0 ? 0 : min(p.splits, (seen + p.chunk - 1) / p.chunk);
        join_row<T, WAVES, 256>(p, parts, wave, n, n == 0, [&](int i) { return i * all + row; }, out);
    }
}

int check(const sptmm_attention_args *a)
{
    if (!a) return fail(SPTMM_ERR_INVALID, "null pointer");
    if (a->type != SPTMM_X_F16 && a->type != SPTMM_X_BF16) return fail(SPTMM_ERR_INVALID, "type must be SPTMM_X_F16 or SPTMM_X_BF16");
    if (a->batch < 0 || a->total_q < 0 || a->max_q < 0 || a->max_kv < 0 || a->kv_rows < 0) return fail(SPTMM_ERR_INVALID, "batch, total_q, max_q, max_kv and kv_rows must not be negative");
    if (a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads || a->q_heads > 65535)
        return fail(SPTMM_ERR_INVALID, "q_heads must be a positive multiple of kv_heads, at most 65535");
    if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8) return fail(SPTMM_ERR_INVALID, "head_dim must be a multiple of 8, 8..256");
    if (!(a->scale > 0.f) || !(a->scale < 1e30f)) return fail(SPTMM_ERR_INVALID, "scale must be positive and below 1e30");
    if ((int64_t)a->total_q * a->q_heads > (1 << 29) || (int64_t)a->batch * a->kv_heads > (1 << 22))  // (2^32 work-items to a launch)
        return fail(SPTMM_ERR_INVALID, "total_q * q_heads must be at most 2^29, batch * kv_heads at most 2^22");
    if (a->kv_rows > (1 << 30)) return fail(SPTMM_ERR_INVALID, "kv_rows must be at most 2^30");
    return SPTMM_OK;
}

// how a call is cut up: by its sizes alone
struct Cut {
    bool keys;  // the KEYS form
    bool stream;
    int dp, slots, splits, chunk, shares, log_rows;
    int most_splits;  // of a call with these sizes and any max_kv up to this one
};
Cut cut(const sptmm_attention_args *a)
{
    Cut c{};
    const int group = a->q_heads / a->kv_heads;
    c.dp = a->head_dim <= 64 ? 64 : a->head_dim <= 128 ? 128 : 256;
    c.keys = (int64_t)a->max_q * group <= 32;
    const int tm = c.keys ? 32 : TILE_ROWS;
    const int64_t rows = (int64_t)a->total_q * group;
    c.slots = (int)(rows / tm + a->batch);
    // workgroups of one tile each (those that have rows): about as many as sequences have tiles
    const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(c.slots, c.keys ? (int64_t)a->batch : rows / tm + 1)) * a->kv_heads;
    const int max_kv = (int)std::min<int64_t>(a->max_kv, a->kv_rows);
    c.splits = c.most_splits = 1;
    if ((int64_t)a->total_q * a->q_heads >= (1 << 24)) {
        // (one launch of the join holds fewer rows)
    } else if (c.keys) {
        // Splits where these are fewer than the chip has places for, two per compute unit.
        const int unit = 128;  // keys a workgroup should have at least
        const int64_t want = (512 + tiles - 1) / tiles, most = (max_kv + unit - 1) / unit;
        c.splits = c.most_splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 256));
        c.chunk = std::max(unit, (max_kv / c.splits + 127) / 128 * 128);
        c.splits = std::max(1, std::min(c.splits, (int)((max_kv + (int64_t)c.chunk - 1) / c.chunk)));
    } else {
        // Shares instead of a workgroup per tile where there are too few tiles to fill the chip evenly.  Heads of 128, bf16: four chunks
        // of 130 to 250 tokens against 12000 to 20000, 5 heads (140 tiles): shares 182 us, tiles 345; eight of 400 against 1400 to 20000
        // (400 tiles) 340 and 385; eight of 300 against 9000, 32 heads (480) 389 and 361; sixteen of 512 against 12000 (960) 629 and
        // 607.  Where the queries are most of the keys tiles see half of theirs, and shares are less equal: 4096 tokens, 1 head of a
        // group of 4 (129) 55 and 69, 3000 tokens, 2 heads (188) 67 and 55, 2000 tokens (126) 45 and 38.
        // Tiles of 256 rows, a workgroup per compute unit, read the keys half as often: one chunk of 161 tokens against 60000 135 us, of
        // 128 rows 157; they are left to work that fills them (200 tokens against 2000: 31 and 25).  A share of two blocks at
        // least: 64 tokens against 1500 18.9 us, of four 22.0.
        const bool chunks = 4ll * a->max_q < max_kv;
        if (tiles < (chunks ? 448 : 160) && max_kv > (chunks ? 512 : 2048)) {
            const int64_t shares = (int64_t)c.slots * a->kv_heads * ((max_kv >> LOG_BLOCK) + 1) / LEAST_BLOCKS;
            c.log_rows = c.dp == 256 || shares < MOST_SHARES ? 7 : 8;
            c.shares = (int)std::min<int64_t>(c.dp == 256 || c.log_rows == 8 ? 256 : MOST_SHARES, (shares + 7) / 8 * 8);
        }
    }
    // Caches that no level below holds between two calls are read past them: 661 MB 120 us (5.5 TB/s), through them 133; 246 MB 55
    // and 61.  Below, no way wins: 123 MB 33.8 and 35.9, 33 MB 14.3 and 13.6.
    c.stream = (int64_t)a->batch * max_kv * a->kv_heads * a->head_dim * 4 > (128ll << 20);
    return c;
}

// rows of parts in the workspace
int64_t part_rows(const sptmm_attention_args *a, const Cut &c) { return c.shares ? 2ll * c.shares << c.log_rows : c.splits > 1 ? (int64_t)a->total_q * a->q_heads * c.splits : 0; }
size_t part_bytes(const sptmm_attention_args *a, const Cut &c) { return ((size_t)part_rows(a, c) * a->head_dim * 4 + 255) / 256 * 256; }
size_t workspace(const sptmm_attention_args *a, const Cut &c) { return part_bytes(a, c) + (size_t)part_rows(a, c) * 8; }

template <int T, int DP, int KT> void launch_tiles(const AttnParams &p, hipStream_t st)
{
    if (p.shares && p.log_rows == 8) {
        if constexpr (DP <= 128) hipLaunchKernelGGL((attention_tile_kernel<T, DP, KT, 8, true>), dim3(p.shares), dim3(512), 0, st, p);
    } else if (p.shares) hipLaunchKernelGGL((attention_tile_kernel<T, DP, KT, 4, true>), dim3(p.shares), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attention_tile_kernel<T, DP, KT, 4, false>), dim3((unsigned)p.slots * p.kv_heads), dim3(256), 0, st, p);
}
template <int T, bool SHARED> void launch_join(const AttnParams &p, bool many, hipStream_t st)
{
    if (many) hipLaunchKernelGGL((attention_join_kernel<T, 4, SHARED>), dim3((unsigned)(p.total_q * p.q_heads)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attention_join_kernel<T, 1, SHARED>), dim3((unsigned)((p.total_q * p.q_heads + 3) / 4)), dim3(256), 0, st, p);
}
template <int T> void launch(const AttnParams &p, const Cut &c, hipStream_t st)
{
    if (c.keys) {
        const dim3 grid(c.slots, p.kv_heads, c.splits);
        const auto kernel = c.dp == 64    ? (c.stream ? attention_keys_kernel<T, 64, 2, true> : attention_keys_kernel<T, 64, 2, false>)
                            : c.dp == 128 ? (c.stream ? attention_keys_kernel<T, 128, 2, true> : attention_keys_kernel<T, 128, 2, false>)
                                          : (c.stream ? attention_keys_kernel<T, 256, 2, true> : attention_keys_kernel<T, 256, 2, false>);
        hipLaunchKernelGGL(kernel, grid, dim3(128), 0, st, p);
        if (c.splits > 1) launch_join<T, false>(p, c.splits > 8, st);
        return;
    }
    if (c.dp == 64) launch_tiles<T, 64, 64>(p, st);
    else if (c.dp == 128) launch_tiles<T, 128, 64>(p, st);
    else launch_tiles<T, 256, 32>(p, st);
    if (c.shares) launch_join<T, true>(p, c.shares > 8ll * (p.total_q * (int64_t)p.group / TILE_ROWS + 1) * p.kv_heads, st);
}

}  // namespace
}  // namespace sptmm

using namespace sptmm;

extern "C" size_t sptmm_attention_workspace_bytes(const sptmm_attention_args *a)
{
    if (check(a) || a->batch == 0 || a->total_q == 0) return 0;
    Cut c = cut(a);
    c.splits = c.most_splits;  // (a little longer cache can have fewer splits, of more keys each)
    return workspace(a, c);
}

extern "C" int sptmm_attention(const sptmm_attention_args *a, void *workspace_dev, size_t workspace_bytes, void *stream)
{
    if (int rc = check(a)) return rc;
    if (a->batch == 0 || a->total_q == 0) return SPTMM_OK;
    if (!a->q || !a->out || !a->q_start || (a->kv_rows > 0 && (!a->k || !a->v))) return fail(SPTMM_ERR_INVALID, "null pointer");
    if ((a->kv_start == nullptr) != (a->kv_len == nullptr)) return fail(SPTMM_ERR_INVALID, "kv_start and kv_len are given together or not at all");
    const int64_t q_row = (int64_t)a->q_heads * a->head_dim, kv_row = (int64_t)a->kv_heads * a->head_dim;
    if (a->q_stride < q_row || a->out_stride < q_row || a->k_stride < kv_row || a->v_stride < kv_row) return fail(SPTMM_ERR_INVALID, "a row stride is shorter than its row of heads");
    if (a->k_stride > (1 << 22) || a->v_stride > (1 << 22)) return fail(SPTMM_ERR_INVALID, "k_stride and v_stride must be at most 2^22 elements");
    if ((a->q_stride | a->k_stride | a->v_stride) % 8 || a->out_stride % 4) return fail(SPTMM_ERR_INVALID, "q, k and v row strides must be multiples of 8 elements, out's of 4");
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) & 15 || (uintptr_t)a->out & 7) return fail(SPTMM_ERR_INVALID, "q, k and v must be aligned to 16 bytes, out to 8");
    if (((uintptr_t)a->q_start | (uintptr_t)a->kv_start | (uintptr_t)a->kv_len) & 3) return fail(SPTMM_ERR_INVALID, "q_start, kv_start and kv_len must be aligned to 4 bytes");
    const Cut c = cut(a);
    const size_t want = workspace(a, c);
    if (want && (!workspace_dev || workspace_bytes < want)) return fail(SPTMM_ERR_INVALID, "the workspace has %zu bytes, %zu are needed", workspace_dev ? workspace_bytes : (size_t)0, want);
    if (want && (uintptr_t)workspace_dev & 15) return fail(SPTMM_ERR_INVALID, "the workspace must be aligned to 16 bytes");
    AttnParams p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.out = a->out;
    p.q_stride = a->q_stride, p.k_stride = a->k_stride, p.v_stride = a->v_stride, p.out_stride = a->out_stride, p.kv_rows = a->kv_rows;
    p.q_start = a->q_start, p.kv_start = a->kv_start, p.kv_len = a->kv_len;
    p.batch = a->batch, p.total_q = a->total_q, p.q_heads = a->q_heads, p.kv_heads = a->kv_heads, p.group = a->q_heads / a->kv_heads, p.dim = a->head_dim;
    p.c = a->scale * 1.44269504088896340736f;
    p.slots = c.slots, p.splits = c.splits, p.chunk = c.chunk, p.shares = c.shares, p.log_rows = c.log_rows;
    p.part_o = (float *)workspace_dev;
    p.part_ml = want ? (float2 *)((char *)workspace_dev + part_bytes(a, c)) : nullptr;
    a->type == SPTMM_X_F16 ? launch<SPTMM_X_F16>(p, c, (hipStream_t)stream) : launch<SPTMM_X_BF16>(p, c, (hipStream_t)stream);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPTMM_OK : fail(SPTMM_ERR_HIP, "attention kernels launch: %s (%d)", hipGetErrorString(e), (int)e);
}
