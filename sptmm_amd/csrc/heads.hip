// What lies between a decoder layer's q+k+v projection and its attention, in one pass: norms of the query and key heads,
// the rotation by position, the rounding to 16 bits, and the scatter of key and value heads to their cache rows.
//
//   x' = x * rsqrt(mean(x^2) + eps) * gain              (query and key heads; without a gain: x' = x)
//   (a, b) -> (a cos w - b sin w, b cos w + a sin w)      pair j of the first 2 * pairs elements, w = position * frequency_j
//
// The angle is kept as a fraction of a turn in 64-bit fixed point: turns_j = frequency_j / 2 pi as a fraction of 2^64, and
// position * turns_j mod 2^64 is the phase, right to position * 2^-65 turns however far the position, of which the upper 32 bits
// are used -- no table of sines to read, and no loss at far positions, where a product in 32 bits is off by position * 2^-24 radians.
// Everything is computed in 32 bits and rounded once, to nearest even, on the way out.
//
// The pass is bound by its bytes: 4096 tokens, 20 + 5 + 5 heads of 128, float in, bf16 out, 94 MB in 18.8 us (5.0 TB/s);
// 20011 tokens, 32 + 8 + 8 heads of 64, fp16, 246 MB in 50 us (4.9 TB/s); a large copy reaches 5.1.  A lane holds four pairs (eight elements: two loads of 16 bytes from float rows), so a
// head of 128 takes 16 lanes and a wavefront handles four heads at a time; the sines of a token's four pairs stay in the
// lane's registers while it walks the token's heads.
#include <cmath>
#include <type_traits>

#include "internal.hpp"
#include "lanes.hpp"

namespace sptmm {
namespace {

typedef unsigned short u16;
typedef __attribute__((ext_vector_type(4))) unsigned short u16x4;
typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

struct HeadsParams {
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride, v_out_stride, kv_capacity;
    const int *positions, *kv_rows;
    const float *q_gain, *k_gain;
    float eps, inv_dim;
    int tokens, q_heads, kv_heads, heads, dim, pairs;  // heads: query + key + value heads of a token (value heads only where v is given)
    int log_lanes;                                     // 1 << log_lanes lanes per head
    int parts, per_part;                               // a token's heads are shared by `parts` wavefronts, `per_part` heads each
    uint64_t turns[SPTMM_MAX_ROTATED_PAIRS];
};

template <int T> __device__ __forceinline__ float widen(u16 b)
{
    if constexpr (T == SPTMM_X_F16) return (float)__builtin_bit_cast(_Float16, b);
    return __builtin_bit_cast(float, (unsigned)b << 16);
}
template <int T> __device__ __forceinline__ u16 narrow(float x)
{
    if constexpr (T == SPTMM_X_F16) return __builtin_bit_cast(u16, (_Float16)x);
    return __builtin_bit_cast(u16, (__bf16)x);
}

// element index of the first (w = 0) and second (w = 1) element of pair slot s
template <bool INTER> __device__ __forceinline__ int element(const HeadsParams &p, int s, int w)
{
    if (INTER) return 2 * s + w;
    const int rest = p.dim / 2 - p.pairs;  // the elements behind the rotated ones are held as pairs too, at angle 0
    return s < p.pairs ? s + w * p.pairs : 2 * p.pairs + (s - p.pairs) + w * rest;
}

// a lane's eight elements as they lie in memory
template <int IN> struct Raw {
    typedef typename std::conditional<IN == SPTMM_X_F32, f32x4, u16x4>::type Run;
    typedef typename std::conditional<IN == SPTMM_X_F32, float, u16>::type One;
    Run a, b;
    static __device__ __forceinline__ float value(One x)
    {
        if constexpr (IN == SPTMM_X_F32) return x;
        else return widen<IN>(x);
    }
};

// four consecutive pair slots from s0 on: two runs of four elements (apart; neighbouring pairs: one run of eight)
template <int IN, bool INTER, bool WIDE> __device__ __forceinline__ void fetch8(const HeadsParams &p, const void *row, int s0, int slots, Raw<IN> &r)
{
    typedef typename Raw<IN>::One One;
    typedef typename Raw<IN>::Run Run;
    const One *const x = (const One *)row;
    if constexpr (WIDE) {
        if constexpr (INTER && IN != SPTMM_X_F32) {
            const u16x8 ab = *reinterpret_cast<const u16x8 *>(x + 2 * s0);
            r.a = __builtin_shufflevector(ab, ab, 0, 1, 2, 3), r.b = __builtin_shufflevector(ab, ab, 4, 5, 6, 7);
        } else {
            r.a = *reinterpret_cast<const Run *>(x + (INTER ? 2 * s0 : element<INTER>(p, s0, 0)));
            r.b = *reinterpret_cast<const Run *>(x + (INTER ? 2 * s0 + 4 : element<INTER>(p, s0, 1)));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // (held as the wide loads would hold them)
            const int sa = INTER ? s0 + i / 2 : s0 + i, sb = INTER ? s0 + 2 + i / 2 : s0 + i;
            r.a[i] = sa < slots ? x[element<INTER>(p, sa, INTER ? i & 1 : 0)] : One(0);
            r.b[i] = sb < slots ? x[element<INTER>(p, sb, INTER ? i & 1 : 1)] : One(0);
        }
    }
}
template <int IN, bool INTER> __device__ __forceinline__ void unpack8(const Raw<IN> &r, float (&x)[2][4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[0][i] = Raw<IN>::value(INTER ? (i < 2 ? r.a[2 * i] : r.b[2 * i - 4]) : r.a[i]);
        x[1][i] = Raw<IN>::value(INTER ? (i < 2 ? r.a[2 * i + 1] : r.b[2 * i - 3]) : r.b[i]);
    }
}

template <int OUT, bool INTER, bool WIDE> __device__ __forceinline__ void store8(const HeadsParams &p, u16 *row, int s0, int slots, const float (&x)[2][4])
{
    if constexpr (WIDE) {
        const int e0 = INTER ? 2 * s0 : element<INTER>(p, s0, 0), e1 = INTER ? 2 * s0 + 4 : element<INTER>(p, s0, 1);
        u16x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = narrow<OUT>(INTER ? x[i & 1][i / 2] : x[0][i]);
            b[i] = narrow<OUT>(INTER ? x[i & 1][2 + i / 2] : x[1][i]);
        }
        if constexpr (INTER) {
            *reinterpret_cast<u16x8 *>(row + e0) = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            *reinterpret_cast<u16x4 *>(row + e0) = a;
            *reinterpret_cast<u16x4 *>(row + e1) = b;
        }
    } else {
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (s0 + i < slots) row[element<INTER>(p, s0 + i, w)] = narrow<OUT>(x[w][i]);
    }
}

// Sine and cosine of the angle that position * turns / 2^64 is a fraction of a turn of.  The phase is cut to its upper 32 bits, more
// than a float holds; the nearest quarter turn is taken off them as an integer, and what is left, an eighth of a turn either
// way (rounded to 24 bits, by 2^-28 of a turn at most), goes into the Taylor polynomials up to x^9 and x^8 (off by 2^-29 and 2^-25 at the ends).
__device__ __forceinline__ void turn(int position, unsigned turns_hi, unsigned turns_lo, float &sine, float &cosine)
{
    const unsigned pos = (unsigned)position;
    unsigned phase = pos * turns_hi + __umulhi(pos, turns_lo);
    if (position < 0) phase -= turns_lo;
    const unsigned quarter = (phase + 0x20000000u) >> 30;
    const float x = (float)(int)(phase - (quarter << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float z = x * x;
    const float s = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.75573192e-6f, -1.98412698e-4f), 8.33333333e-3f), -1.66666667e-1f), 1.0f);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.48015873e-5f, -1.38888889e-3f), 4.16666667e-2f), -0.5f), 1.0f);
    const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
    sine = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, a) ^ (quarter & 2) << 30);
    cosine = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, b) ^ ((quarter + 1) & 2) << 30);
}

// Rounds of heads whose loads a wavefront has in flight together.  4096 tokens, 20 + 5 + 5 heads of 128, float in: two 18.8 us, one
// or four 19.7; 20011 tokens, 32 + 8 + 8 heads of 64, fp16 in: two 50, one 53, four 56 (registers that more wavefronts use better).
constexpr int ROUNDS = 2;

// IN: type of the rows; OUT: type of the heads written; INTER: pairs of neighbours (2j, 2j+1), else of halves (j, j + pairs);
// WIDE: every run of four elements lies aligned for one load or store
template <int IN, int OUT, bool INTER, bool WIDE> __global__ void __launch_bounds__(256) heads_kernel(const HeadsParams p)
{
    const int lane = threadIdx.x & 63;
    const int per_wave = 64 >> p.log_lanes, sub = lane >> p.log_lanes, s0 = (lane & ((1 << p.log_lanes) - 1)) * 4, slots = p.dim / 2;
    const bool mine = s0 < slots;
    // the lane's frequencies and gains
    unsigned t_hi[4], t_lo[4];
    float gq[2][4], gk[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t x = s0 + i < p.pairs ? p.turns[s0 + i] : 0;
        t_hi[i] = (unsigned)(x >> 32), t_lo[i] = (unsigned)x;
    }
    {
        Raw<SPTMM_X_F32> g, h;
        g.a = g.b = h.a = h.b = f32x4{1.f, 1.f, 1.f, 1.f};
        if (p.q_gain && mine) fetch8<SPTMM_X_F32, INTER, WIDE>(p, p.q_gain, s0, slots, g);
        if (p.k_gain && mine) fetch8<SPTMM_X_F32, INTER, WIDE>(p, p.k_gain, s0, slots, h);
        unpack8<SPTMM_X_F32, INTER>(g, gq);
        unpack8<SPTMM_X_F32, INTER>(h, gk);
    }
    const int64_t units = (int64_t)p.tokens * p.parts;
    for (int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += (int64_t)gridDim.x * 4) {
        const int t = p.parts == 1 ? (int)unit : (int)(unit / p.parts), part = (int)(unit - (int64_t)t * p.parts);
        const int first = part * p.per_part, end = min(p.heads, first + p.per_part);
        const int pos = p.positions ? p.positions[t] : t;
        const int64_t kv_row = p.kv_rows ? p.kv_rows[t] : t;
        const bool kept = kv_row >= 0 && kv_row < p.kv_capacity;
        constexpr int ESZ = IN == SPTMM_X_F32 ? 4 : 2;
        float cs[4], sn[4];
        bool ready = false;
        for (int h0 = first; h0 < end; h0 += ROUNDS * per_wave) {
            // the loads of all rounds first
            Raw<IN> raw[ROUNDS];
#pragma unroll
            for (int u = 0; u < ROUNDS; ++u) {
                const int h = h0 + u * per_wave + sub;
                const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
                const int at = is_q ? h : is_v ? h - p.q_heads - p.kv_heads : h - p.q_heads;
                const char *src = (const char *)(is_q ? p.q : is_v ? p.v : p.k) + ((int64_t)t * (is_q ? p.q_stride : is_v ? p.v_stride : p.k_stride) + (int64_t)at * p.dim) * ESZ;
                if (mine && h < end) fetch8<IN, INTER, WIDE>(p, src, s0, slots, raw[u]);
                else raw[u].a = raw[u].b = typename Raw<IN>::Run{0, 0, 0, 0};
            }
            if (!ready) {  // the token's sines, while the loads are on their way
                ready = true;
#pragma unroll
                for (int i = 0; i < 4; ++i) turn(pos, t_hi[i], t_lo[i], sn[i], cs[i]);
            }
#pragma unroll
            for (int u = 0; u < ROUNDS; ++u) {
                const int h = h0 + u * per_wave + sub;
                if (h - sub >= end) break;
                const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
                const int at = is_q ? h : is_v ? h - p.q_heads - p.kv_heads : h - p.q_heads;
                float x[2][4];
                unpack8<IN, INTER>(raw[u], x);
                if (p.q_gain || p.k_gain) {
                    float sum = 0.f;
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum = fmaf(x[w][i], x[w][i], sum);
                    if (p.log_lanes >= 2) sum = lanes_sum(sum, p.log_lanes);
                    else if (p.log_lanes == 1) sum += dpp<0xB1>(sum);  // quad_perm [1,0,3,2]
                    if (!is_v && (is_q ? p.q_gain : p.k_gain)) {  // (lanes of one head agree)
                        const float r = rsqrtf(fmaf(sum, p.inv_dim, p.eps));
#pragma unroll
                        for (int w = 0; w < 2; ++w)
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[w][i] = x[w][i] * r * (is_q ? gq[w][i] : gk[w][i]);
                    }
                }
                if (!is_v)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (s0 + i < p.pairs) {
                            const float a = x[0][i], b = x[1][i];
                            x[0][i] = a * cs[i] - b * sn[i];
                            x[1][i] = b * cs[i] + a * sn[i];
                        }
                if (mine && h < end && (is_q || kept)) {
                    u16 *dst = (u16 *)(is_q ? p.q_out : is_v ? p.v_out : p.k_out) +
                               ((is_q ? (int64_t)t * p.q_out_stride : kv_row * (is_v ? p.v_out_stride : p.k_out_stride)) + (int64_t)at * p.dim);
                    store8<OUT, INTER, WIDE>(p, dst, s0, slots, x);
                }
            }
        }
    }
}

template <int IN, int OUT> void launch_in_out(const HeadsParams &p, bool inter, bool wide, int blocks, hipStream_t st)
{
    const auto kernel = inter ? (wide ? heads_kernel<IN, OUT, true, true> : heads_kernel<IN, OUT, true, false>)
                              : (wide ? heads_kernel<IN, OUT, false, true> : heads_kernel<IN, OUT, false, false>);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, p);
}

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace
}  // namespace sptmm

using namespace sptmm;

extern "C" int sptmm_rotation_init(const double *radians_per_position, int pairs, int interleaved, sptmm_rotation *out)
{
    if (!out || (pairs > 0 && !radians_per_position)) return fail(SPTMM_ERR_INVALID, "null pointer");
    if (pairs < 0 || pairs > SPTMM_MAX_ROTATED_PAIRS) return fail(SPTMM_ERR_INVALID, "pairs must be 0..%d", SPTMM_MAX_ROTATED_PAIRS);
    sptmm_rotation r{};
    r.pairs = pairs;
    r.interleaved = interleaved ? 1 : 0;
    for (int j = 0; j < pairs; ++j) {
        const long double turn = (long double)radians_per_position[j] / 6.283185307179586476925286766559005768L;
        if (!std::isfinite((double)turn)) return fail(SPTMM_ERR_INVALID, "the frequency of pair %d is not finite", j);
        const long double whole = floorl(turn), f = (turn - whole) * 18446744073709551616.0L;  // fraction of a turn, of 2^64
        r.turns[j] = f >= 18446744073709551615.0L ? UINT64_MAX : (uint64_t)(f + 0.5L);
    }
    *out = r;
    return SPTMM_OK;
}

extern "C" int sptmm_heads_norm_rotate(const sptmm_heads_args *a, void *stream)
{
    if (!a) return fail(SPTMM_ERR_INVALID, "null pointer");
    if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->q_heads + a->kv_heads < 1 || a->q_heads > 65535 || a->kv_heads > 65535)
        return fail(SPTMM_ERR_INVALID, "tokens, q_heads and kv_heads must not be negative, at most 65535 heads, and not both counts zero");
    if (a->head_dim < 2 || a->head_dim > 256 || a->head_dim % 2) return fail(SPTMM_ERR_INVALID, "head_dim must be even, 2..256");
    if (a->in_type != SPTMM_X_F16 && a->in_type != SPTMM_X_BF16 && a->in_type != SPTMM_X_F32)
        return fail(SPTMM_ERR_INVALID, "in_type must be SPTMM_X_F16, SPTMM_X_BF16 or SPTMM_X_F32");
    if (a->out_type != SPTMM_X_F16 && a->out_type != SPTMM_X_BF16) return fail(SPTMM_ERR_INVALID, "out_type must be SPTMM_X_F16 or SPTMM_X_BF16");
    if (a->tokens == 0) return SPTMM_OK;
    const bool has_v = a->v != nullptr;
    if ((a->q_heads && (!a->q || !a->q_out)) || (a->kv_heads && (!a->k || !a->k_out)) || (a->kv_heads && has_v && !a->v_out))
        return fail(SPTMM_ERR_INVALID, "null pointer");
    const int64_t q_row = (int64_t)a->q_heads * a->head_dim, kv_row = (int64_t)a->kv_heads * a->head_dim;
    if (a->q_stride < q_row || a->q_out_stride < q_row || a->k_stride < kv_row || a->k_out_stride < kv_row ||
        (has_v && (a->v_stride < kv_row || a->v_out_stride < kv_row)))
        return fail(SPTMM_ERR_INVALID, "a row stride is shorter than its row of heads");
    if (a->kv_capacity < 0) return fail(SPTMM_ERR_INVALID, "kv_capacity must not be negative");
    const sptmm_rotation *rot = a->rotation;
    if (rot && (rot->pairs < 0 || rot->pairs > SPTMM_MAX_ROTATED_PAIRS || 2 * rot->pairs > a->head_dim))
        return fail(SPTMM_ERR_INVALID, "the rotation has %d pairs, more than half of head_dim %d", rot->pairs, a->head_dim);
    if ((a->q_gain || a->k_gain) && !(a->eps >= 0.f && a->eps < 1e30f)) return fail(SPTMM_ERR_INVALID, "eps must be finite and not negative");
    // elements and their natural alignment
    const size_t isz = a->in_type == SPTMM_X_F32 ? 4 : 2;
    const void *ins[3] = {a->q, a->k, a->v}, *outs[3] = {a->q_out, a->k_out, a->v_out}, *words[4] = {a->positions, a->kv_rows, a->q_gain, a->k_gain};
    for (const void *x : ins)
        if (!aligned(x, isz)) return fail(SPTMM_ERR_INVALID, "rows must be aligned to their elements");
    for (const void *x : outs)
        if (!aligned(x, 2)) return fail(SPTMM_ERR_INVALID, "rows must be aligned to their elements");
    for (const void *x : words)
        if (!aligned(x, 4)) return fail(SPTMM_ERR_INVALID, "positions, kv_rows and gains must be aligned to 4 bytes");

    HeadsParams p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out, p.k_out = a->k_out, p.v_out = a->v_out;
    p.q_stride = a->q_stride, p.k_stride = a->k_stride, p.v_stride = a->v_stride;
    p.q_out_stride = a->q_out_stride, p.k_out_stride = a->k_out_stride, p.v_out_stride = a->v_out_stride;
    p.kv_capacity = a->kv_capacity;
    p.positions = a->positions, p.kv_rows = a->kv_rows, p.q_gain = a->q_gain, p.k_gain = a->k_gain;
    p.eps = a->eps, p.inv_dim = 1.0f / (float)a->head_dim;
    p.tokens = a->tokens, p.q_heads = a->q_heads, p.kv_heads = a->kv_heads, p.dim = a->head_dim;
    p.heads = a->q_heads + a->kv_heads * (has_v ? 2 : 1);
    const bool inter = rot && rot->interleaved;
    if (rot) {
        p.pairs = rot->pairs;
        for (int j = 0; j < rot->pairs; ++j) p.turns[j] = rot->turns[j];
    }
    p.log_lanes = 0;
    while ((8 << p.log_lanes) < a->head_dim) ++p.log_lanes;
    const int per_wave = 64 >> p.log_lanes, rounds = (p.heads + per_wave - 1) / per_wave;
    // One wavefront per round of heads while that leaves the chip's wavefront slots unfilled (a lone token: one round of
    // latency instead of eight); one per token once there are enough tokens (its sines are computed once).  20 + 5 + 5 heads of
    // 128, a wavefront per round and one per token: 64 tokens 7.4 us and 8.4, 512 7.7 and 9.2, 1024 9.4 and 10.0, 1500 11.6 and 11.0,
    // 4096 27 and 19.
    p.parts = a->tokens >= 1024 ? 1 : rounds;
    const int rounds_per_part = (rounds + p.parts - 1) / p.parts;
    p.per_part = rounds_per_part * per_wave;
    const int64_t units = (int64_t)a->tokens * p.parts;
    const int blocks = (int)std::min<int64_t>((units + 3) / 4, 1 << 22);

    // runs of four elements aligned for one load / store: in the head (dim, pairs) and from row to row
    const size_t in4 = inter && isz == 2 ? 16 : 4 * isz, out4 = inter ? 16 : 8;
    bool wide = a->head_dim % 8 == 0 && (inter || p.pairs % 4 == 0);
    const int64_t strides[6] = {a->q_stride, a->k_stride, has_v ? a->v_stride : 0, a->q_out_stride, a->k_out_stride, has_v ? a->v_out_stride : 0};
    for (int64_t s : strides) wide = wide && s % (inter ? 8 : 4) == 0;
    for (const void *x : ins) wide = wide && aligned(x, in4);
    for (const void *x : outs) wide = wide && aligned(x, out4);
    wide = wide && aligned(a->q_gain, 16) && aligned(a->k_gain, 16);

    hipStream_t st = (hipStream_t)stream;
    const bool h = a->out_type == SPTMM_X_F16;
    switch (a->in_type) {
    case SPTMM_X_F16: h ? launch_in_out<SPTMM_X_F16, SPTMM_X_F16>(p, inter, wide, blocks, st) : launch_in_out<SPTMM_X_F16, SPTMM_X_BF16>(p, inter, wide, blocks, st); break;
    case SPTMM_X_BF16: h ? launch_in_out<SPTMM_X_BF16, SPTMM_X_F16>(p, inter, wide, blocks, st) : launch_in_out<SPTMM_X_BF16, SPTMM_X_BF16>(p, inter, wide, blocks, st); break;
    default: h ? launch_in_out<SPTMM_X_F32, SPTMM_X_F16>(p, inter, wide, blocks, st) : launch_in_out<SPTMM_X_F32, SPTMM_X_BF16>(p, inter, wide, blocks, st); break;
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPTMM_OK : fail(SPTMM_ERR_HIP, "heads_kernel launch: %s (%d)", hipGetErrorString(e), (int)e);
}
