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
// Two forms.  TILE (prompts): the wavefronts of a workgroup take 32 rows each and share tiles of 64 keys.  KEYS (single
// tokens: all rows of a tile fit one wavefront's 32): every wavefront takes its own tiles of 32 keys.  Either may split the
// keys over workgroups; unnormalised sums and statistics then go to a workspace and attention_join_kernel adds them up in
// their order.
//
// Rounding: products of 16-bit values summed in 32 bits; statistics, sums and rescaling in 32 bits; p is rounded to 16 bits
// for the second product (half a step of p each, bf16 2^-8 and fp16 2^-11 of it: the terms' errors average out), the result once.
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
    int splits, chunk;
    float *part_o;  // [split][query * q_heads + head][dim], unnormalised
    float2 *part_ml;  // [split][query * q_heads + head]: the maximum that the sums are relative to (of raw scores), sum
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
    __device__ __forceinline__ void init(int64_t stride, int dim, int wave, bool is_v)
    {
        const int lane = threadIdx.x & 63;
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

    __device__ __forceinline__ void init(const AttnParams &p, const Tile &t, int kv_head, int row, bool valid)
    {
        const int lane = threadIdx.x & 63, half = lane >> 5;
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
        // the weights relative to `top`, rounded into pf; their 32-bit sum.  fp16: p is held 2^7 larger, so that what rounds to zero is
        // below 2^-32 of the largest.
        auto weigh = [&] {
            const float at = (top == -INFINITY ? 0.f : top * p.c) - (T == SPTMM_X_F16 ? 7.f : 0.f);
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[b][e], p.c, -at));
                    part[e & 3] += x;
                    pf[2 * b + (e >> 3)][e & 7] = narrow<T>(x);
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

template <int T> __device__ __forceinline__ void write4(const AttnParams &p, const Tile &t, int kv_head, int row, int d, int split, f32x4 x)
{
    const int i = row / p.group, head = kv_head * p.group + row - i * p.group;
    if (p.splits > 1) {
        *reinterpret_cast<f32x4 *>(p.part_o + ((int64_t)split * p.total_q * p.q_heads + (int64_t)(t.q0 + i) * p.q_heads + head) * p.dim + d) = x;
        return;
    }
    u16x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = narrow<T>(x[e]);
    *reinterpret_cast<u16x4 *>(p.out + (int64_t)(t.q0 + i) * p.out_stride + (int64_t)head * p.dim + d) = y;
}

// ------------------------------------------------------------------------------------------------ TILE: rows over wavefronts
// Bound by the matrix units' feed: one prompt of 8192 tokens, 20 heads of 128 on 5, bf16: 344 GFLOP in 325 to 345 us, 1.0 to 1.06 PFLOP/s, where a
// product of two 8192 x 8192 matrices reaches 1.21 on the same card.  64 KB of LDS leave two workgroups to a compute unit, and
// one's exponentials run beside the other's products; of the time, the exponentials alone are a tenth, the loads 3 %.  Four
// wavefronts of 32 rows share each tile of K and V through the LDS (without bank conflicts); of 256 rows: slower, one workgroup a unit.
template <int T, int DP, int KT, int WAVES> __global__ void __launch_bounds__(64 * WAVES, DP == 256 ? 1 : 2) attention_tile_kernel(const AttnParams p)
{
    static_assert(WAVES == 4, "128 rows");
    constexpr int LOG_TM = 7, TM = 1 << LOG_TM;
    __shared__ __attribute__((aligned(1024))) char k_a[KT * DP * 2], k_b[KT * DP * 2], v_a[KT * DP * 2], v_b[KT * DP * 2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    // A sequence's last rows, which see the most keys, first, and of all heads before the next rows: workgroups dispatched late
    // are short.  (All sequences' tiles in one order of the keys they see: eight chunks of up to 400 tokens 361 us, so 371; thirty
    // prompts of 30 to 1500 tokens 170, so 150.  Heads kept to their XCDs' L2s: one prompt of 8192, 5 heads, 341 and 346; 32 heads 524 and 510.)
    const int kv_head = (int)(blockIdx.x % (unsigned)p.kv_heads), split = blockIdx.z, slot = p.slots - 1 - (int)(blockIdx.x / (unsigned)p.kv_heads);
    if (!find_tile<LOG_TM>(p, slot, &t)) return;
    const int i_last = (min(t.row0 + TM, t.rows) - 1) / p.group, all = min(t.nk, t.nk - t.nq + i_last + 1);
    const int begin = split * p.chunk, end = split == p.splits - 1 ? all : min(all, begin + p.chunk);
    if (split && begin >= end) return;

    Loader<DP, KT, WAVES> lk, lv;
    lk.init(p.k_stride, p.dim, wave, false);
    lv.init(p.v_stride, p.dim, wave, true);
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
    r.init(p, t, kv_head, valid ? row : t.rows - 1, valid);
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
    const float sum = halves_sum(r.sum), f = p.splits > 1 ? 1.f : 1.f / sum;
    if (!valid) return;
    const bool none = r.lim < 0;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = 32 * d + 8 * e + 4 * (lane >> 5);
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = none ? 0.f : r.o[d][4 * e + i] * f;
            if (at < p.dim) write4<T>(p, t, kv_head, row, at, split, x);
        }
    if (p.splits > 1 && lane < 32) {
        const int i = row / p.group, head = kv_head * p.group + row - i * p.group;
        p.part_ml[(int64_t)split * p.total_q * p.q_heads + (int64_t)(t.q0 + i) * p.q_heads + head] = float2{r.top, sum};
    }
}

// ------------------------------------------------------------------------------------------------ KEYS: keys over wavefronts
// Bound by the cache's read: 32 sequences of 2000 to 8000 keys, 661 MB, 5.5 TB/s.  Nothing is shared between wavefronts but the
// sums at the end, so that each waits for its own loads only.  Two to a workgroup, as 128 KB of LDS for four leave one workgroup
// to a compute unit: 20 heads of 128 on 5, one token against 8000 keys 13.7 us and 18.6, 32 against 1500 36 and 40, 64: 55 and 54.
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
    lk.init(p.k_stride, p.dim, 0, false);
    lv.init(p.v_stride, p.dim, 0, true);
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
    r.init(p, t, kv_head, t.row0 + (valid ? lane & 31 : 0), valid);
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
    // the wavefronts' sums, brought to one maximum and added in wavefront order; a wavefront's part lies where its tiles lay
    const float sum = halves_sum(r.sum);
    if (lane < 32) tops[wave][lane] = r.top, sums[wave][lane] = sum;
    __syncthreads();
    float top = tops[0][lane & 31];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, tops[w][lane & 31]);
    const float f = r.top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((r.top - top) * p.c);
    constexpr int PER = ONE / 4096;  // blocks of 32 values of d that one array has room for
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = r.top == -INFINITY ? 0.f : r.o[d][4 * e + i] * f;
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
        for (int w = 0; w < WAVES; ++w) total += tops[w][rr] == -INFINITY ? 0.f : sums[w][rr] * __builtin_amdgcn_exp2f((tops[w][rr] - best) * p.c);
        const int row = t.row0 + rr, i = row / p.group;
        if (p.splits > 1) {
            if (d4 == 0)
                p.part_ml[(int64_t)split * p.total_q * p.q_heads + (int64_t)(t.q0 + i) * p.q_heads + kv_head * p.group + row - i * p.group] = float2{best, total};
        } else {
            const float inv = 1.f / total;
            const bool none = t.nk - t.nq + i < 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = none ? 0.f : x[c] * inv;
        }
        write4<T>(p, t, kv_head, row, 4 * d4, split, x);
    }
}

// ------------------------------------------------------------------------------------------------ splits joined
// Per (query, head) the splits that hold keys the row sees, added in a fixed order, by WAVES wavefronts: the four of a workgroup
// where there are many splits (one token of 20 heads against 8000 keys, 63 splits: the call 13.6 us, by single wavefronts
// 16.8), one where there are few and many rows (870 x 20 rows of four: 204 us, by four wavefronts each 217).
template <int T, int WAVES> __global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p)
{
    __shared__ __attribute__((aligned(16))) f32x4 parts[4][64];
    const int lane = threadIdx.x & 63, in_block = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = WAVES == 1 ? 0 : in_block;
    const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + in_block : blockIdx.x, all = (int64_t)p.total_q * p.q_heads;
    if (row >= all) return;
    const int query = (int)(row / p.q_heads), head = (int)(row - (int64_t)query * p.q_heads);
    // the sequence of this query: the last one that starts at or before it
    Seq s = {0, 0, 0, 0};
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const int b = b0 + lane;
        const Seq mine = sequence(p, min(b, p.batch - 1));
        const int c = __popcll(__ballot(b < p.batch && mine.q0 <= query));
        if (c == 0) break;
        s = {__builtin_amdgcn_readlane(mine.q0, c - 1), __builtin_amdgcn_readlane(mine.nq, c - 1), 0, __builtin_amdgcn_readlane(mine.nk, c - 1)};
        if (c < 64) break;
    }
    if (query >= s.q0 + s.nq) return;  // a row behind the last sequence
    const int seen = s.nk - s.nq + (query - s.q0) + 1;
    const int n = seen <= 0 ? 0 : min(p.splits, (seen + p.chunk - 1) / p.chunk);
    // every lane holds the weight of one split (and of those 64, 128 and 192 further)
    float2 ml[4];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ml[i] = lane + 64 * i < n ? p.part_ml[(lane + 64 * i) * all + row] : float2{-INFINITY, 0.f};
        top = fmaxf(top, ml[i].x);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[i].x - top) * p.c);
        sum = fmaf(ml[i].y, w[i], sum);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    // four values a lane, and as many splits side by side as lanes are left, and every WAVES-th such group a wavefront's
    const int quads = p.dim / 4, log_l = quads <= 2 ? 1 : 32 - __builtin_clz(quads - 1), sub = lane >> log_l, d4 = lane & ((1 << log_l) - 1), step = 64 >> log_l;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int end = min(64, n - 64 * i);
        for (int s0 = wave * step; s0 < end; s0 += 4 * WAVES * step) {
            f32x4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {  // (four loads in flight; behind the last split: its values, times zero)
                const int at = min(64 * i + s0 + u * WAVES * step + sub, n - 1);
                x[u] = *reinterpret_cast<const f32x4 *>(p.part_o + (at * all + row) * p.dim + 4 * min(d4, quads - 1));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int at = s0 + u * WAVES * step + sub;
                const float f = __shfl(w[i], at & 63, 64);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = at < end ? fmaf(x[u][e], f, o[e]) : o[e];
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
    for (int e = 0; e < 4; ++e) y[e] = narrow<T>(n ? o[e] * inv : 0.f);
    *reinterpret_cast<u16x4 *>(p.out + (int64_t)query * p.out_stride + (int64_t)head * p.dim + 4 * d4) = y;
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
    int dp, slots, splits, chunk;
};

Cut cut(const sptmm_attention_args *a)
{
    Cut c{};
    const int group = a->q_heads / a->kv_heads;
    c.dp = a->head_dim <= 64 ? 64 : a->head_dim <= 128 ? 128 : 256;
    c.keys = (int64_t)a->max_q * group <= 32;
    const int tm = c.keys ? 32 : 128;
    const int64_t rows = (int64_t)a->total_q * group;
    c.slots = (int)(rows / tm + a->batch);
    // Workgroups without splits (those that have rows): about as many as sequences have tiles.  Splits where they are fewer than
    // the chip has places for -- two per compute unit, of the TILE form with heads of 256 one --, in the TILE form three quarters
    // of that: 512 tokens against 16000 keys, 8 heads: 113 us, with all the places 134; eight chunks of 64 tokens against 3000
    // to 9000, 5 heads: 67 and 75; four chunks of 130 to 250 against 12000 to 20000, 5 heads: 214 and 200.
    const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(c.slots, c.keys ? (int64_t)a->batch : rows / tm + 1)) * a->kv_heads;
    const int64_t room = c.keys ? 512 : c.dp == 256 ? 192 : 384;
    const int max_kv = (int)std::min<int64_t>(a->max_kv, a->kv_rows);
    // Keys a workgroup should have at least.  Where the queries are most of the keys, half the tiles see little of a late split
    // and the join has many rows: one prompt of 600, 1024, 1500 tokens, 20 heads on 5: 19, 25, 35 us at 2048, 27, 32, 48 at 512
    // (2000 tokens, 8 heads on 2: 40 and 36).  A chunk of 64 against 1500, of 200 against 2000: 32, 41 us at 2048, 21, 25 at 512.
    const int unit = c.keys ? 128 : 2ll * a->max_q >= max_kv ? 2048 : 512;
    const int64_t want = (room + tiles - 1) / tiles, most = (max_kv + unit - 1) / unit;
    c.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 256));
    if ((int64_t)a->total_q * a->q_heads >= (1 << 24)) c.splits = 1;  // (one launch of the join holds fewer rows)
    c.chunk = std::max(unit, (max_kv / c.splits + 127) / 128 * 128);
    c.splits = std::max(1, std::min(c.splits, (max_kv + c.chunk - 1) / c.chunk));
    // Caches that no level below holds between two calls are read past them: 661 MB 120 us (5.5 TB/s), through them 133; 246 MB 55
    // and 61.  Below, no way wins: 123 MB 33.8 and 35.9, 33 MB 14.3 and 13.6.
    c.stream = (int64_t)a->batch * max_kv * a->kv_heads * a->head_dim * 4 > (128ll << 20);
    return c;
}

size_t workspace(const sptmm_attention_args *a, const Cut &c)
{
    if (c.splits <= 1) return 0;
    const size_t rows = (size_t)a->total_q * a->q_heads * c.splits;
    return (rows * a->head_dim * 4 + 255) / 256 * 256 + rows * 8;
}

template <int T> void launch(const AttnParams &p, const Cut &c, hipStream_t st)
{
    const dim3 grid = c.keys ? dim3(c.slots, p.kv_heads, c.splits) : dim3((unsigned)c.slots * p.kv_heads, 1, c.splits);
    if (c.keys) {
        const auto kernel = c.dp == 64    ? (c.stream ? attention_keys_kernel<T, 64, 2, true> : attention_keys_kernel<T, 64, 2, false>)
                            : c.dp == 128 ? (c.stream ? attention_keys_kernel<T, 128, 2, true> : attention_keys_kernel<T, 128, 2, false>)
                                          : (c.stream ? attention_keys_kernel<T, 256, 2, true> : attention_keys_kernel<T, 256, 2, false>);
        hipLaunchKernelGGL(kernel, grid, dim3(128), 0, st, p);
    } else {
        if (c.dp == 64) hipLaunchKernelGGL((attention_tile_kernel<T, 64, 64, 4>), grid, dim3(256), 0, st, p);
        else if (c.dp == 128) hipLaunchKernelGGL((attention_tile_kernel<T, 128, 64, 4>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((attention_tile_kernel<T, 256, 32, 4>), grid, dim3(256), 0, st, p);
    }
    if (c.splits <= 1) return;
    if (c.splits > 8) hipLaunchKernelGGL((attention_join_kernel<T, 4>), dim3((unsigned)(p.total_q * p.q_heads)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attention_join_kernel<T, 1>), dim3((unsigned)((p.total_q * p.q_heads + 3) / 4)), dim3(256), 0, st, p);
}

}  // namespace
}  // namespace sptmm

using namespace sptmm;

extern "C" size_t sptmm_attention_workspace_bytes(const sptmm_attention_args *a)
{
    if (check(a) || a->batch == 0 || a->total_q == 0) return 0;
    return workspace(a, cut(a));
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
    p.slots = c.slots, p.splits = c.splits, p.chunk = c.chunk;
    p.part_o = (float *)workspace_dev;
    const size_t o_bytes = ((size_t)a->total_q * a->q_heads * c.splits * a->head_dim * 4 + 255) / 256 * 256;
    p.part_ml = want ? (float2 *)((char *)workspace_dev + o_bytes) : nullptr;
    a->type == SPTMM_X_F16 ? launch<SPTMM_X_F16>(p, c, (hipStream_t)stream) : launch<SPTMM_X_BF16>(p, c, (hipStream_t)stream);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPTMM_OK : fail(SPTMM_ERR_HIP, "attention kernels launch: %s (%d)", hipGetErrorString(e), (int)e);
}
