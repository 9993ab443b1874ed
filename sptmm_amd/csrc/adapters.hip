// Low-rank adapters of many requests beside one shared projection:
//
//   Y[m][n] = base[m][n] + scale_s * sum_r B_s[n][r] * h[m][r],   h[m][r] = sum_k A_s[r][k] X[m][k],   s = row_slot[m]
//
// In general two launches.  The first makes h: 16 rows of X against 16 ranks of A per matrix instruction (16-bit operands, 32-bit
// sums), the rows' contraction over K split over wavefronts and workgroups.  The second adds up the splits' partial sums in
// their order and multiplies by B on the 32-bit matrix instruction: h is never rounded to 16 bits -- outputs are 32-bit
// floats, and a rounded h would cost them fifteen of their bits -- and B's 16-bit values are exact in 32.  (Many rows: on the 16-bit
// instruction, by exact parts of both.)
//
// Rows come in any order of slots.  A tile of 16 rows is walked once per distinct slot in it (found by ballots, no sorting
// pass); a matrix column is a row of X and stays in its lanes throughout, so rows of other slots are left out by a select
// and never by a product with zero: an infinity in one adapter's weights reaches its own rows only.
//
// Both weights sit in the order in which a wavefront reads them, 1 KiB per load instruction (adapters_pack_kernel).
//
// Many rows are bound by base, Y and X: 3001 rows, K=2560 N=13824, eight slots of rank 16 to 64: 356 MB in 101 us (fp16 107), 3.5 TB/s (an
// addition to an array of that size, 332 MB, 57 us).  A few rows are bound by latency: one row 6.7 to 8.6 us where an empty launch
// takes 3.5; 48 rows of 32 slots, K=6912 N=2560: 18 MB in 13 to 15.5 us, two launches that each wait for slots, weights and sums.
#include <cmath>

#include "internal.hpp"
#include "lanes.hpp"

namespace sptmm {
// What the kernels know of a slot.
struct alignas(16) SlotInfo {
    int rank;  // 0: empty
    float scale;
    int bad;  // B holds a value that is not finite
};
}  // namespace sptmm

struct sptmm_adapters {
    int K, N, type, slots, max_rank;
    int k_steps;     // steps of 32 along K (the last one padded with zeros)
    int n_pairs;     // pairs of 16 columns
    int max_chunks;  // chunks of 16 ranks a slot has room for
    int device, compute_units;
    uint16_t *A, *B;  // [slot]: [chunk][k_step][64 lanes][8] and [n_pair][chunk][64 lanes][8], packed by the chunks in use
    sptmm::SlotInfo *info;
};

namespace sptmm {
namespace {

typedef unsigned short u16;
typedef __attribute__((ext_vector_type(4))) unsigned short u16x4;
typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

template <int T> __device__ __forceinline__ f32x4 mfma16(u16x8 a, u16x8 b, f32x4 c)
{
    if constexpr (T == SPTMM_X_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int T> __device__ __forceinline__ float widen(u16 b)
{
    if constexpr (T == SPTMM_X_F16) return (float)__builtin_bit_cast(_Float16, b);
    return __builtin_bit_cast(float, (unsigned)b << 16);
}

struct AdapterArgs {
    const u16 *X, *A, *B;
    const int *row_slot;
    const SlotInfo *info;
    const float *base;
    float *h, *Y;
    int M, K, N, slots, k_steps, n_pairs, max_chunks, tiles, splits, places;
};

// ------------------------------------------------------------------------------------------------ weights into place
// The slot's info, by a launch of its own before the weights': a captured set clears the mark anew with every replay.
__global__ void adapters_info_kernel(SlotInfo *info, int rank, float scale) { *info = SlotInfo{rank, scale, 0}; }

// One thread per stored value.  A lane of the first product's operand holds rank lane % 16, k = 8 * (lane / 16) + e of a step
// of 32; of the second's, column lane % 16 (e < 4) or 16 + lane % 16 (e >= 4) of a pair, rank 4 * (lane / 16) + e % 4 of a chunk.
__global__ void __launch_bounds__(256) adapters_pack_kernel(const u16 *A, const u16 *B, u16 *pA, u16 *pB, SlotInfo *info, int rank, int K, int N, int k_steps, int n_pairs,
                                                            int chunks, unsigned exponent)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t na = (int64_t)chunks * k_steps * 512, nb = (int64_t)n_pairs * chunks * 512;
    const int e = (int)(i & 7), lane = (int)(i >> 3) & 63;
    if (i < na) {
        const int step = (int)((i >> 9) % k_steps), c = (int)((i >> 9) / k_steps);
        const int r = 16 * c + (lane & 15), k = 32 * step + 8 * (lane >> 4) + e;
        const u16 x = r < rank && k < K ? A[(int64_t)r * K + k] : (u16)0;
        pA[i] = x;
    }
    if (i < nb) {
        const int c = (int)((i >> 9) % chunks), pair = (int)((i >> 9) / chunks);
        const int n = 32 * pair + 16 * (e >> 2) + (lane & 15), r = 16 * c + 4 * (lane >> 4) + (e & 3);
        const u16 x = r < rank && n < N ? B[(int64_t)n * rank + r] : (u16)0;
        pB[i] = x;
        if ((x & exponent) == exponent) info->bad = 1;
    }
}

// the distinct slots of the rows that the low 16 lanes hold: call with the mask of rows not yet served
__device__ __forceinline__ int next_slot(int slot, unsigned long long &left)
{
    const int s = __builtin_amdgcn_readlane(slot, __builtin_ctzll(left));
    left &= ~__ballot(slot == s);
    return s;
}

__device__ __forceinline__ int chunks_of(int rank) { return (rank + 15) >> 4; }

// slot of the row that this lane holds (row tile * 16 + lane % 16), -1 where it has none
__device__ __forceinline__ int slot_of(const AdapterArgs &p, int m)
{
    const int s = m < p.M ? p.row_slot[m] : -1;
    return s >= 0 && s < p.slots ? s : -1;
}

// ------------------------------------------------------------------------------------------------ h = X A^T
constexpr int SHRINK_WAVES = 8;
constexpr int CHUNKS_AT_ONCE = 4;  // chunks of 16 ranks summed in one walk over K (X is read once per walk)
constexpr int STEPS_AT_ONCE = 4;   // steps of 32 along K whose loads are in flight together

// this wavefront's share of NC chunks' sums over the steps step0, step0 + SHRINK_WAVES, ... below step1
template <int T, int NC> __device__ __forceinline__ void walk_k(const AdapterArgs &p, const u16 *a, const u16 *x_row, int step0, int step1, f32x4 (&acc)[CHUNKS_AT_ONCE])
{
    const int k_lane = 8 * ((threadIdx.x & 63) >> 4);
    for (int step = step0; step < step1; step += STEPS_AT_ONCE * SHRINK_WAVES) {
        u16x8 x[STEPS_AT_ONCE], w[STEPS_AT_ONCE][NC];
#pragma unroll
        for (int u = 0; u < STEPS_AT_ONCE; ++u) {
            const int at = min(step + u * SHRINK_WAVES, step1 - 1);
            x[u] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (32 * at + k_lane < p.K) x[u] = *reinterpret_cast<const u16x8 *>(x_row + 32 * at);
#pragma unroll
            for (int c = 0; c < NC; ++c) w[u][c] = *reinterpret_cast<const u16x8 *>(a + ((int64_t)c * p.k_steps + at) * 512);
        }
#pragma unroll
        for (int u = 0; u < STEPS_AT_ONCE; ++u)
            if (step + u * SHRINK_WAVES < step1)
#pragma unroll
                for (int c = 0; c < NC; ++c) acc[c] = mfma16<T>(w[u][c], x[u], acc[c]);
    }
}

// chunks c0 .. c0 + nc - 1 of slot s, summed over a range of K by the workgroup's eight wavefronts: afterwards wavefront w < nc
// holds chunk c0 + w of all 16 rows.  The wavefronts' shares are added through the LDS in wavefront order.
template <int T> __device__ __forceinline__ f32x4 shrink(const AdapterArgs &p, f32x4 (&sums)[SHRINK_WAVES][CHUNKS_AT_ONCE][64], int s, int rank, int c0, int nc, const u16 *x_row, int step0, int step1)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f32x4 acc[CHUNKS_AT_ONCE];
#pragma unroll
    for (int c = 0; c < CHUNKS_AT_ONCE; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u16 *a = p.A + ((int64_t)s * p.max_chunks + c0) * p.k_steps * 512 + lane * 8;
    switch (nc) {
    case 1: walk_k<T, 1>(p, a, x_row, step0 + wave, step1, acc); break;
    case 2: walk_k<T, 2>(p, a, x_row, step0 + wave, step1, acc); break;
    case 3: walk_k<T, 3>(p, a, x_row, step0 + wave, step1, acc); break;
    default: walk_k<T, 4>(p, a, x_row, step0 + wave, step1, acc); break;
    }
#pragma unroll
    for (int c = 0; c < CHUNKS_AT_ONCE; ++c)
        if (c < nc) sums[wave][c][lane] = acc[c];
    __syncthreads();
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    if (wave < nc) {
        t = sums[0][wave][lane];
#pragma unroll
        for (int w = 1; w < SHRINK_WAVES; ++w) t += sums[w][wave][lane];
        // ranks that only fill up the chunk: zeros whatever X holds (its infinities times their zeros are none)
        const int r = 16 * (c0 + wave) + 4 * (lane >> 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = r + e < rank ? t[e] : 0.f;
    }
    return t;
}

// Workgroup (tile of 16 rows, split of K, group of four chunks and place among the tile's distinct slots): it serves every
// `places`-th distinct slot of the tile.
template <int T> __global__ void __launch_bounds__(SHRINK_WAVES * 64) adapters_shrink_kernel(const AdapterArgs p)
{
    __shared__ __attribute__((aligned(16))) f32x4 sums[SHRINK_WAVES][CHUNKS_AT_ONCE][64];
    const int tile = blockIdx.x, split = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = (int)(blockIdx.z / p.places) * CHUNKS_AT_ONCE, place = (int)(blockIdx.z % p.places);
    const int m = tile * 16 + (lane & 15), slot = slot_of(p, m);
    unsigned long long left = __ballot(slot >= 0) & 0xffff;
    const int per = (p.k_steps + p.splits - 1) / p.splits, step0 = split * per, step1 = min(p.k_steps, step0 + per);
    const u16 *x_row = p.X + (int64_t)min(m, p.M - 1) * p.K + 8 * (lane >> 4);
    for (int o = 0; left; ++o) {
        const int s = next_slot(slot, left);
        if (o % p.places != place) continue;
        const int rank = p.info[s].rank, nc = min(CHUNKS_AT_ONCE, chunks_of(rank) - c0);
        if (nc <= 0) continue;
        const f32x4 t = shrink<T>(p, sums, s, rank, c0, nc, x_row, step0, step1);
        if (wave < nc && slot == s) reinterpret_cast<f32x4 *>(p.h)[(((int64_t)split * p.tiles + tile) * p.max_chunks + c0 + wave) * 64 + lane] = t;
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ Y = base + scale * h B^T
// 16 rows x 32 columns of one chunk of 16 ranks, on the 32-bit matrix instruction; rows that do not use the slot keep y
template <int T> __device__ __forceinline__ void add_chunk(u16x8 b, f32x4 h, bool mine, f32x4 &y0, f32x4 &y1)
{
    f32x4 n0 = y0, n1 = y1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        n0 = __builtin_amdgcn_mfma_f32_16x16x4f32(widen<T>(b[e]), h[e], n0, 0, 0, 0);
        n1 = __builtin_amdgcn_mfma_f32_16x16x4f32(widen<T>(b[4 + e]), h[e], n1, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y0[e] = mine ? n0[e] : y0[e], y1[e] = mine ? n1[e] : y1[e];
}
// The same on the 16-bit matrix instruction: where many rows make the second product long enough to stand beside its bytes.  A
// 32-bit h is the sum of three parts of bf16, exactly and whatever its size (from 2^-102 on: no part is subnormal); a bf16 value of B
// is one part, an fp16 value (11 bits, of the range of bf16) the sum of two.  Every part of B meets every part of h, two pairs of parts sharing an instruction's
// 32 places along the contraction: two instructions to 16 columns (bf16) or three, each an eighth of the 32-bit way's time.  No bit of
// the inner sums is lost: a small one beside a large one that the column does not use counts in full.  An h that is not
// finite is its first part, and stays away from B's second one (infinity times that part's zeros is none of the product); a
// B that is not finite goes the 32-bit way.
template <int T> struct Parts {
    u16x8 h12, h31, h23;  // parts of h, by the pairs that an instruction takes (bf16: the first two; the upper half of h31 is zero)

    static __device__ __forceinline__ unsigned top_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0xffff0000u; }
    __device__ __forceinline__ void split(f32x4 h)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = h[e];
            const bool finite = fabsf(x) < INFINITY;
            const unsigned hi = top_bits(x);
            const float r = finite ? x - __builtin_bit_cast(float, hi) : 0.f;
            const unsigned mid = top_bits(r);
            const u16 one = (u16)(hi >> 16), two = (u16)(mid >> 16), three = (u16)(top_bits(r - __builtin_bit_cast(float, mid)) >> 16);
            h12[e] = one, h12[4 + e] = two, h31[e] = three, h31[4 + e] = T == SPTMM_X_F16 && finite ? one : (u16)0;
            if constexpr (T == SPTMM_X_F16) h23[e] = two, h23[4 + e] = three;
        }
    }
    // 16 columns: x holds four ranks' values of B
    __device__ __forceinline__ f32x4 columns(u16x4 x, f32x4 y) const
    {
        if constexpr (T == SPTMM_X_F16) {
            u16x8 b;  // its two parts
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = widen<T>(x[e]);
                const unsigned hi = top_bits(v);
                b[e] = (u16)(hi >> 16), b[4 + e] = (u16)(__builtin_bit_cast(unsigned, v - __builtin_bit_cast(float, hi)) >> 16);
            }
            return mfma16<SPTMM_X_BF16>(b, h31, mfma16<SPTMM_X_BF16>(b, h23, mfma16<SPTMM_X_BF16>(b, h12, y)));
        } else {
            const u16x8 b = __builtin_shufflevector(x, x, 0, 1, 2, 3, 0, 1, 2, 3);
            return mfma16<T>(b, h31, mfma16<T>(b, h12, y));
        }
    }
    __device__ __forceinline__ void add_chunk(u16x8 b, bool mine, f32x4 &y0, f32x4 &y1) const
    {
        const f32x4 n0 = columns(__builtin_shufflevector(b, b, 0, 1, 2, 3), y0), n1 = columns(__builtin_shufflevector(b, b, 4, 5, 6, 7), y1);
#pragma unroll
        for (int e = 0; e < 4; ++e) y0[e] = mine ? n0[e] : y0[e], y1[e] = mine ? n1[e] : y1[e];
    }
};
// the operand of column pair `pair`, chunk c of slot s (`chunks` chunks in use)
__device__ __forceinline__ u16x8 load_b(const AdapterArgs &p, int s, int pair, int chunks, int c)
{
    return *reinterpret_cast<const u16x8 *>(p.B + ((int64_t)s * p.n_pairs * p.max_chunks + (int64_t)pair * chunks + c) * 512 + (threadIdx.x & 63) * 8);
}

// A wavefront takes one tile of 16 rows and CP pairs of 16 columns.  The four wavefronts of a workgroup take neighbouring columns
// of one tile or (ROWS) the same columns of four tiles: few rows need many workgroups, and many rows are bound by base and Y, of
// which a wavefront then moves 512 bytes of every row.  The rows' h (each row its own slot's) is first brought into the LDS,
// scaled and with the splits' partial sums added in their order; then the distinct slots are walked.
// Without ROWS the distinct slots of a tile are shared by `places` workgroups, which write the rows of their own.
template <int T, int CP, bool ROWS> __global__ void __launch_bounds__(256) adapters_expand_kernel(const AdapterArgs p)
{
    extern __shared__ __attribute__((aligned(16))) f32x4 h_lds[];  // [ROWS ? 4 : 1][max_chunks][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = (ROWS ? 1 : 4) * CP, groups = (p.n_pairs + per - 1) / per;
    const int tile = (int)(blockIdx.x / groups) * (ROWS ? 4 : 1) + (ROWS ? wave : 0);
    const int pair = (int)(blockIdx.x % groups) * per + (ROWS ? 0 : wave * CP);
    const int m = tile * 16 + (lane & 15), slot = slot_of(p, m);
    unsigned long long left = __ballot(slot >= 0) & 0xffff;
    bool write = m < p.M;
    if (!ROWS && p.places > 1) {  // the slots of this workgroup's place, and for the first place the rows without a slot
        unsigned long long rest = left;
        left = 0;
        for (int o = 0; rest; ++o) {
            const unsigned long long before = rest;
            next_slot(slot, rest);
            if (o % p.places == (int)blockIdx.z) left |= before & ~rest;
        }
        if (!left && blockIdx.z) return;
        write = write && (slot >= 0 ? (left >> (lane & 15) & 1) != 0 : blockIdx.z == 0);
    }
    const int64_t at = (int64_t)m * p.N + pair * 32 + 4 * (lane >> 4);
    const int cols = (p.N - pair * 32) / 16;  // groups of 16 columns from here on
    f32x4 acc[CP][2];
#pragma unroll
    for (int c = 0; c < CP; ++c)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            acc[c][g] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (p.base && write && 2 * c + g < cols) acc[c][g] = *reinterpret_cast<const f32x4 *>(p.base + at + 32 * c + 16 * g);
        }
    // the walk's place: DEEP chunks from c on of slot s (s < 0: the walk is over); its first B is on its way while h is brought in
    constexpr int DEEP = ROWS ? 1 : 4;
    struct Place {
        int s, chunks, c;
    };
    auto after = [&](Place at) {
        if ((at.c += DEEP) < at.chunks) return at;
        at.c = 0;
        do {
            at.s = left ? next_slot(slot, left) : -1;
            at.chunks = at.s >= 0 ? chunks_of(p.info[at.s].rank) : 0;
        } while (at.s >= 0 && at.chunks == 0);
        return at;
    };
    auto load = [&](const Place &at, u16x8(&b)[DEEP][CP]) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
#pragma unroll
            for (int i = 0; i < CP; ++i)
                if (at.s >= 0 && 2 * i < cols) b[d][i] = load_b(p, at.s, pair + i, at.chunks, min(at.c + d, at.chunks - 1));
    };
    Place now = after(Place{-1, 0, 0});
    u16x8 b[DEEP][CP];
    load(now, b);

    const SlotInfo mine = slot >= 0 && write ? p.info[slot] : SlotInfo{0, 0.f, 0};
    const int my_chunks = chunks_of(mine.rank);
    const unsigned long long wide = __ballot(mine.rank && mine.bad);  // rows whose B takes the 32-bit instruction
    f32x4 *const h_tile = h_lds + (ROWS ? wave * p.max_chunks * 64 : 0);
    for (int c = ROWS ? 0 : wave; c < p.max_chunks; c += ROWS ? 1 : 4) {
        if (!__ballot(c < my_chunks)) break;
        if (c < my_chunks) {
            const f32x4 *hp = reinterpret_cast<const f32x4 *>(p.h) + ((int64_t)tile * p.max_chunks + c) * 64 + lane;
            const int64_t next = (int64_t)p.tiles * p.max_chunks * 64;
            f32x4 h = hp[0];
            int k = 1;
            for (; k + 4 <= p.splits; k += 4) {
                const f32x4 a = hp[k * next], b = hp[(k + 1) * next], c4 = hp[(k + 2) * next], d = hp[(k + 3) * next];
                h += a, h += b, h += c4, h += d;
            }
            for (; k < p.splits; ++k) h += hp[k * next];
            h *= mine.scale;
            h_tile[c * 64 + lane] = h;
        }
    }
    __syncthreads();
    if (cols <= 0) return;
    Parts<T> parts;
    while (now.s >= 0) {
        const Place then = after(now);
        u16x8 next[DEEP][CP];
        load(then, next);
        const bool serves = slot == now.s, by_parts = ROWS && !(wide & __ballot(serves));
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            if (now.c + d >= now.chunks) break;
            const f32x4 h = h_tile[(now.c + d) * 64 + lane];
            if (by_parts) parts.split(h);
#pragma unroll
            for (int i = 0; i < CP; ++i)
                if (2 * i < cols) {
                    if (by_parts) parts.add_chunk(b[d][i], serves, acc[i][0], acc[i][1]);
                    else add_chunk<T>(b[d][i], h, serves, acc[i][0], acc[i][1]);
                }
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
#pragma unroll
            for (int i = 0; i < CP; ++i) b[d][i] = next[d][i];
        now = then;
    }
#pragma unroll
    for (int c = 0; c < CP; ++c)
#pragma unroll
        for (int g = 0; g < 2; ++g)
            if (write && 2 * c + g < cols) *reinterpret_cast<f32x4 *>(p.Y + at + 32 * c + 16 * g) = acc[c][g];
}

// ------------------------------------------------------------------------------------------------ both products in one launch
// For a row or a few: workgroup (256 columns, tile, ordinal of a distinct slot) computes its rows' h whole -- every workgroup of a
// slot reads all of A, which costs less than a second launch while A is small -- and multiplies it by its columns of B.
template <int T> __global__ void __launch_bounds__(SHRINK_WAVES * 64) adapters_fused_kernel(const AdapterArgs p)
{
    __shared__ __attribute__((aligned(16))) f32x4 sums[SHRINK_WAVES][CHUNKS_AT_ONCE][64], h_lds[CHUNKS_AT_ONCE][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = blockIdx.x * SHRINK_WAVES + wave;
    const int m = blockIdx.y * 16 + (lane & 15), slot = slot_of(p, m);
    unsigned long long left = __ballot(slot >= 0) & 0xffff;
    for (int o = blockIdx.z; o > 0 && left; --o) next_slot(slot, left);
    if (!left && blockIdx.z) return;
    const int s = left ? __builtin_amdgcn_readlane(slot, __builtin_ctzll(left)) : -2, rank = left ? p.info[s].rank : 0, chunks = chunks_of(rank);
    const bool write = m < p.M && (slot == s || (blockIdx.z == 0 && slot < 0));
    const int n0 = pair * 32 + 4 * (lane >> 4);
    const bool first = pair < p.n_pairs, second = pair * 32 + 16 < p.N;
    const int64_t at = (int64_t)m * p.N + n0;
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (p.base && write && first) acc[0] = *reinterpret_cast<const f32x4 *>(p.base + at);
    if (p.base && write && second) acc[1] = *reinterpret_cast<const f32x4 *>(p.base + at + 16);
    const float scale = chunks ? p.info[s].scale : 0.f;
    const u16 *x_row = p.X + (int64_t)min(m, p.M - 1) * p.K + 8 * (lane >> 4);
    for (int c0 = 0; c0 < chunks; c0 += CHUNKS_AT_ONCE) {
        const int nc = min(CHUNKS_AT_ONCE, chunks - c0);
        u16x8 b[CHUNKS_AT_ONCE];
        if (first)
#pragma unroll
            for (int c = 0; c < CHUNKS_AT_ONCE; ++c) b[c] = load_b(p, s, pair, chunks, min(c0 + c, chunks - 1));
        const f32x4 t = shrink<T>(p, sums, s, rank, c0, nc, x_row, 0, p.k_steps);
        if (wave < nc) h_lds[wave][lane] = t * scale;
        __syncthreads();
        if (first)
#pragma unroll
            for (int c = 0; c < CHUNKS_AT_ONCE; ++c)
                if (c < nc) add_chunk<T>(b[c], h_lds[c][lane], slot == s, acc[0], acc[1]);
    }
    if (write && first) *reinterpret_cast<f32x4 *>(p.Y + at) = acc[0];
    if (write && second) *reinterpret_cast<f32x4 *>(p.Y + at + 16) = acc[1];
}

// (the runtime keeps a failed call's error until it is asked for: taken here, or the next launch would be blamed for it)
int hip_fail(hipError_t e, const char *what)
{
    (void)hipGetLastError();
    return e == hipErrorOutOfMemory ? fail(SPTMM_ERR_NOMEM, "%s: out of device memory", what) : fail(SPTMM_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

// One tile of rows, and A small (KiB of the largest slot, and of all workgroups' reads if every row has another slot): both
// products run in one launch.  K=2560 N=3840, one row: rank 32 (160 KiB) 8.1 us, in two launches 11.2; rank 64 (320) 8.3 and 10.8;
// rank 128 (640) 13.4 and 11.1.  Sixteen rows of sixteen slots of rank 16: N=3840 (19 MiB) 8.1 and 10.7, N=13824 (68) 19.9 and 13.0;
// eight rows (34) 10.7 both ways.
constexpr int FUSED_A_KIB = 320, FUSED_READ_KIB = 32 << 10;

bool fused(const sptmm_adapters *a, int M)
{
    const int64_t kib = (int64_t)a->max_chunks * a->k_steps, groups = (a->n_pairs + SHRINK_WAVES - 1) / SHRINK_WAVES;
    return M <= 16 && kib <= FUSED_A_KIB && kib * groups * M <= FUSED_READ_KIB;
}

// Workgroups that share the distinct slots of a tile.  Decode: every row may have another slot, and a workgroup that walks sixteen
// waits for sixteen chains of loads; prompts: a tile rarely has more than two, and workgroups that find none cost their launch.
// K=2560 N=3840, ranks 16 to 32, one, four or sixteen places: 64 rows of 64 slots 48, 22, 17 us; 256 rows of 64 slots 58, 36, 47;
// 256 rows of prompts of 8 slots 13.5, 11.7, 14.0; 3001 rows, N=13824: 104, 101, 109.
int places_of(int M) { return M < 16 ? M : M <= 128 ? 16 : 4; }

// splits of K over workgroups: enough of them to fill the chip, each wavefront with two steps of 32 at least
int splits_of(const sptmm_adapters *a, int M)
{
    const int tiles = (M + 15) / 16, groups = tiles * (M <= 128 ? places_of(M) : 1);
    const int want = (a->compute_units + groups - 1) / groups, most = (a->k_steps + 2 * SHRINK_WAVES - 1) / (2 * SHRINK_WAVES);
    return want < 1 ? 1 : want < most ? want : most;
}

size_t need(const sptmm_adapters *a, int M)
{
    return fused(a, M) ? 0 : (size_t)splits_of(a, M) * ((M + 15) / 16) * a->max_chunks * 64 * 16;
}

// The most that any call of up to M rows needs: fewer rows have more splits, and 4080 rows can need twice what 4096 do.  From as many
// tiles as compute units on there is one split, and the need grows with the rows.
size_t most_need(const sptmm_adapters *a, int M)
{
    size_t most = need(a, M);
    for (int m = 1; m <= std::min(M, 128); ++m) most = std::max(most, need(a, m));
    for (int m = 144; m <= M && m / 16 <= a->compute_units; m += 16) most = std::max(most, need(a, m));
    return most;
}

int check_device(const sptmm_adapters *a)
{
    int dev = -1;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
    if (dev != a->device) return fail(SPTMM_ERR_INVALID, "the adapters live on device %d but device %d is current", a->device, dev);
    return SPTMM_OK;
}

template <int T> void launch_apply(const AdapterArgs &p, bool one_launch, hipStream_t st)
{
    if (one_launch) {
        hipLaunchKernelGGL((adapters_fused_kernel<T>), dim3((p.n_pairs + SHRINK_WAVES - 1) / SHRINK_WAVES, p.tiles, p.places), dim3(SHRINK_WAVES * 64), 0, st, p);
        return;
    }
    const int groups = (p.n_pairs + 3) / 4, z = p.places * ((p.max_chunks + CHUNKS_AT_ONCE - 1) / CHUNKS_AT_ONCE);
    const size_t lds = (size_t)p.max_chunks * 1024;
    hipLaunchKernelGGL((adapters_shrink_kernel<T>), dim3(p.tiles, p.splits, z), dim3(SHRINK_WAVES * 64), 0, st, p);
    // Fewer workgroups of the many-row kind than this leave compute units idle.  K=2560, ranks 8 to 64 of 32 slots, rows in any order
    // (in prompts), without and with it: 512 x 3840 (240 workgroups) 63, 65 us (16.8, 20.6); 1024 x 2560 (320) 78, 81 (18.9, 21.8);
    // 512 x 6912 (432) 85, 72 (21.8, 22.7); 1024 x 6912 (864) 140, 105 (30.5, 26.6); 3001 x 13824 in prompts 127, 102.  fp16, whose B
    // comes apart on the way: 512 x 6912 83, 86 (23.3, 24.9); 1024 x 6912 140, 129 (34.9, 31.6); 1024 x 13824 243, 194 (60.5, 53.6);
    // 3001 x 13824 in prompts of rank 16 to 64 142, 107, of 64 to 128 196, 161, of 96 to 192 235, 222, and of 128 to 256 288, 349: there
    // the sums of four tiles fill the LDS.
    if ((int64_t)(p.tiles / 4) * groups < 400 || (T == SPTMM_X_F16 && p.max_chunks > 12))
        hipLaunchKernelGGL((adapters_expand_kernel<T, 1, false>), dim3(p.tiles * groups, 1, p.places), dim3(256), lds, st, p);
    else
        hipLaunchKernelGGL((adapters_expand_kernel<T, 4, true>), dim3((p.tiles + 3) / 4 * groups), dim3(256), 4 * lds, st, p);
}

}  // namespace
}  // namespace sptmm

using namespace sptmm;

extern "C" void sptmm_adapters_free(sptmm_adapters *a)
{
    if (!a) return;
    if (a->A) (void)hipFree(a->A);
    if (a->B) (void)hipFree(a->B);
    if (a->info) (void)hipFree(a->info);
    delete a;
}

extern "C" int sptmm_adapters_create(int K, int N, int type, int slots, int max_rank, sptmm_adapters **out)
{
    if (!out) return fail(SPTMM_ERR_INVALID, "null pointer");
    if (K < 16 || N < 16 || K % 16 || N % 16) return fail(SPTMM_ERR_INVALID, "K and N must be positive multiples of 16");
    if (K > (1 << 20) || N > (1 << 20)) return fail(SPTMM_ERR_INVALID, "K and N must be at most 2^20");
    if (type != SPTMM_X_F16 && type != SPTMM_X_BF16) return fail(SPTMM_ERR_INVALID, "type must be SPTMM_X_F16 or SPTMM_X_BF16");
    if (slots < 1 || slots > 65536) return fail(SPTMM_ERR_INVALID, "slots must be 1..65536");
    if (max_rank < 1 || max_rank > 256) return fail(SPTMM_ERR_INVALID, "max_rank must be 1..256");
    sptmm_adapters *a = new (std::nothrow) sptmm_adapters();
    if (!a) return fail(SPTMM_ERR_NOMEM, "out of host memory");
    a->K = K, a->N = N, a->type = type, a->slots = slots, a->max_rank = max_rank;
    a->k_steps = (K + 31) / 32, a->n_pairs = (N + 31) / 32, a->max_chunks = (max_rank + 15) / 16;
    const size_t per_a = (size_t)a->max_chunks * a->k_steps * 1024, per_b = (size_t)a->max_chunks * a->n_pairs * 1024;
    hipError_t e = hipGetDevice(&a->device);
    if (e == hipSuccess) e = hipDeviceGetAttribute(&a->compute_units, hipDeviceAttributeMultiprocessorCount, a->device);
    if (e == hipSuccess) e = hipMalloc((void **)&a->A, per_a * slots);
    if (e == hipSuccess) e = hipMalloc((void **)&a->B, per_b * slots);
    if (e == hipSuccess) e = hipMalloc((void **)&a->info, sizeof(SlotInfo) * slots);
    if (e == hipSuccess) e = hipMemset(a->info, 0, sizeof(SlotInfo) * slots);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        sptmm_adapters_free(a);
        return hip_fail(e, "sptmm_adapters_create");
    }
    *out = a;
    return SPTMM_OK;
}

extern "C" int sptmm_adapters_set(sptmm_adapters *a, int slot, const uint16_t *A, const uint16_t *B, int rank, float scale, void *stream)
{
    if (!a) return fail(SPTMM_ERR_INVALID, "null pointer");
    if (slot < 0 || slot >= a->slots) return fail(SPTMM_ERR_INVALID, "slot %d out of range (have %d)", slot, a->slots);
    if (rank < 0 || rank > a->max_rank) return fail(SPTMM_ERR_INVALID, "rank must be 0 (empty the slot) to %d", a->max_rank);
    if (rank && (!A || !B)) return fail(SPTMM_ERR_INVALID, "null pointer");
    if (!std::isfinite(scale)) return fail(SPTMM_ERR_INVALID, "scale must be finite");
    if (int rc = check_device(a)) return rc;
    const int chunks = (rank + 15) / 16;
    const int64_t n = (int64_t)chunks * 512 * std::max(a->k_steps, a->n_pairs);
    u16 *pA = a->A + (size_t)slot * a->max_chunks * a->k_steps * 512, *pB = a->B + (size_t)slot * a->max_chunks * a->n_pairs * 512;
    hipLaunchKernelGGL(adapters_info_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, a->info + slot, rank, scale);
    if (n)
        hipLaunchKernelGGL(adapters_pack_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, A, B, pA, pB, a->info + slot, rank, a->K, a->N, a->k_steps,
                           a->n_pairs, chunks, a->type == SPTMM_X_F16 ? 0x7c00u : 0x7f80u);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPTMM_OK : hip_fail(e, "adapters_pack_kernel launch");
}

extern "C" size_t sptmm_adapters_workspace_bytes(const sptmm_adapters *a, int M)
{
    if (!a || M < 1) return 0;
    return most_need(a, M);
}

extern "C" int sptmm_adapters_apply(const sptmm_adapters *a, const uint16_t *X, const int32_t *row_slot, int M, const float *base, float *Y, void *workspace,
                                    size_t workspace_bytes, void *stream)
{
    if (!a || !X || !row_slot || !Y) return fail(SPTMM_ERR_INVALID, "null pointer");
    if (M < 1) return fail(SPTMM_ERR_INVALID, "M must be at least 1");
    if (M > (1 << 24)) return fail(SPTMM_ERR_INVALID, "M must be at most 2^24");
    if (((uintptr_t)X | (uintptr_t)base | (uintptr_t)Y | (uintptr_t)workspace) & 15) return fail(SPTMM_ERR_INVALID, "X, base, Y and the workspace must be aligned to 16 bytes");
    if ((uintptr_t)row_slot & 3) return fail(SPTMM_ERR_INVALID, "row_slot must be aligned to 4 bytes");
    const size_t want = need(a, M);
    if (want && (!workspace || workspace_bytes < want))
        return fail(SPTMM_ERR_INVALID, "the workspace has %zu bytes, %zu are needed", workspace ? workspace_bytes : (size_t)0, want);
    // (a dimension of a launch holds 2^32 work-items)
    if ((int64_t)((M + 15) / 16) * ((a->n_pairs + 3) / 4) >= (1 << 24)) return fail(SPTMM_ERR_UNSUPPORTED, "M = %d rows by N = %d columns are more than one launch holds", M, a->N);
    if (int rc = check_device(a)) return rc;
    AdapterArgs p{};
    p.X = X, p.A = a->A, p.B = a->B, p.row_slot = row_slot, p.info = a->info, p.base = base, p.h = (float *)workspace, p.Y = Y;
    p.M = M, p.K = a->K, p.N = a->N, p.slots = a->slots, p.k_steps = a->k_steps, p.n_pairs = a->n_pairs, p.max_chunks = a->max_chunks;
    p.tiles = (M + 15) / 16, p.splits = splits_of(a, M), p.places = places_of(M);
    a->type == SPTMM_X_F16 ? launch_apply<SPTMM_X_F16>(p, fused(a, M), (hipStream_t)stream) : launch_apply<SPTMM_X_BF16>(p, fused(a, M), (hipStream_t)stream);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPTMM_OK : hip_fail(e, "adapters kernels launch");
}
