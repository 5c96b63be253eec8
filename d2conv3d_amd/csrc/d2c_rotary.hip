// Rotary positions along time, height and width: channel pair j of a head turns by position[axis of j] * rate_j, with
// rate = base^(-i / pairs of the axis) for the i-th pair of an axis; the way back is the turn by the opposite angle.
//
// Bound: memory (each value read and written once): 207360 tokens of 8 heads of 64, bfloat16, 78 us (5.4 TB/s, a large copy 5.15); 25920 of 4 heads of 80, float32,
// tensor of positions, 17.5 us (3.8 TB/s, much of it the way to and from a kernel); a single frame's 350, 3.7 us.  A workgroup takes some tokens, works out their cosines and sines once for all
// heads (LDS), then moves the tokens' channels in 16-byte vectors.
// An angle is made in turns, position * rate / 2 pi, with the rate as the sum of two floats (48 bits, made from a base in 64), so that what remains after
// whole turns are taken off is exact to float32 for positions of up to 2^24, where float32 stops to tell whole ones apart; beyond, it is off by position * rate *
// 2^-48 turns.  A product in float32 of a position of 10^4 would be off by 5e-4 radians.
#include <algorithm>
#include <cmath>
#include "d2c_common.hpp"
#include "d2c_mma.hpp"

namespace {

constexpr int kRotThreads = 256, kRotLds = 32 << 10;

struct RotArgs {
    const void *x;
    const float *pos;
    void *y;
    long xs[3], ps;
    int L, H, D, pairs, end0, end1;      // pairs 0 .. end0 - 1 turn with time, .. end1 - 1 with height
    int gh, gw, tokens;                  // the grid's height and width; tokens to a workgroup
    float sign;
    float hi[D2C_ROTARY_MAX_PAIRS], lo[D2C_ROTARY_MAX_PAIRS];      // turns for a position's step
};

template <typename T, bool INTERLEAVED> __global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotArgs a)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ float2 s_cs[];      // [token][pair]
    const int t0 = (int)blockIdx.x * a.tokens, n = (int)blockIdx.y, count = min(a.tokens, a.L - t0);
    for (int i = threadIdx.x; i < count * a.pairs; i += kRotThreads) {
        const int t = i / a.pairs, j = i - t * a.pairs, token = t0 + t, axis = j < a.end0 ? 0 : j < a.end1 ? 1 : 2;
        float p;
        if (a.pos) p = a.pos[n * a.ps + (long)token * 3 + axis];
        else {
            const int line = token / a.gw;
            p = (float)(axis == 2 ? token - line * a.gw : axis == 0 ? line / a.gh : line % a.gh);
        }
        const float part = fmaf(p, a.lo[j], fmaf(p, a.hi[j], -rintf(p * a.hi[j])));      // (the inner one: rounded once, below 1 in size)
        float s, c;
        sincospif(2.f * part, &s, &c);
        s_cs[i] = make_float2(c, s * a.sign);
    }
    __syncthreads();

    // a unit: a vector of pairs (INTERLEAVED: VEC / 2 of them side by side; else VEC of them, their second channels a vector further on), or
    // a vector of channels that pass
    const int turn = INTERLEAVED ? (2 * a.pairs + VEC - 1) / VEC : (a.pairs + VEC - 1) / VEC;
    const int units = turn + (a.D - 2 * a.pairs + VEC - 1) / VEC;
    const T *xb = reinterpret_cast<const T *>(a.x) + n * a.xs[0];
    T *yb = reinterpret_cast<T *>(a.y) + (long)n * a.L * a.H * a.D;
    for (int i = threadIdx.x; i < count * a.H * units; i += kRotThreads) {
        const int line = i / units, u = i - line * units, t = line / a.H, h = line - t * a.H;
        const T *x = xb + (long)(t0 + t) * a.xs[1] + (long)h * a.xs[2];
        T *y = yb + ((long)(t0 + t) * a.H + h) * a.D;
        const float2 *cs = s_cs + t * a.pairs;
        if (u >= turn) {
            const int d = 2 * a.pairs + (u - turn) * VEC;
            store_run<T>(y + d, load_run<T>(x + d, a.D - d), a.D - d);
        } else if constexpr (INTERLEAVED) {
            const int d = u * VEC, left = 2 * a.pairs - d;
            alignas(16) T e[VEC];
            *reinterpret_cast<uint4 *>(e) = load_run<T>(x + d, left);
#pragma unroll
            for (int k = 0; k < VEC; k += 2) {
                const float2 w = cs[min(d + k, 2 * a.pairs - 2) / 2];
                const float p = elem_to_f32<T>(e[k]), q = elem_to_f32<T>(e[k + 1]);
                e[k] = f32_to_elem<T>(p * w.x - q * w.y);
                e[k + 1] = f32_to_elem<T>(p * w.y + q * w.x);
            }
            store_run<T>(y + d, *reinterpret_cast<const uint4 *>(e), left);
        } else {
            const int d = u * VEC, left = a.pairs - d;
            alignas(16) T e[VEC], f[VEC];
            *reinterpret_cast<uint4 *>(e) = load_run<T>(x + d, left);
            *reinterpret_cast<uint4 *>(f) = load_run<T>(x + a.pairs + d, left);
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const float2 w = cs[min(d + k, a.pairs - 1)];
                const float p = elem_to_f32<T>(e[k]), q = elem_to_f32<T>(f[k]);
                e[k] = f32_to_elem<T>(p * w.x - q * w.y);
                f[k] = f32_to_elem<T>(p * w.y + q * w.x);
            }
            store_run<T>(y + d, *reinterpret_cast<const uint4 *>(e), left);
            store_run<T>(y + a.pairs + d, *reinterpret_cast<const uint4 *>(f), left);
        }
    }
}

int check(const d2c_rotary3d_desc *q)
{
    if (!q) { d2c_set_error("rotary: null description"); return D2C_ERR_SHAPE; }
    if (q->dtype != D2C_F32 && q->dtype != D2C_BF16) { d2c_set_error("rotary: float32 or bfloat16 only"); return D2C_ERR_DTYPE; }
    if (q->N < 0 || q->L < 0 || q->H <= 0 || q->D <= 0) { d2c_set_error("rotary: sizes must not be negative, heads and their size positive"); return D2C_ERR_SHAPE; }
    if (q->N > 65535) { d2c_set_error("rotary: too many samples"); return D2C_ERR_SHAPE; }
    if (q->H > (1 << 20) || q->D > (1 << 16) || (long)q->H * q->D > (1L << 24)) { d2c_set_error("rotary: too many channels"); return D2C_ERR_SHAPE; }
    long pairs = 0;
    for (int p : q->pairs) {
        if (p < 0 || p > D2C_ROTARY_MAX_PAIRS) { d2c_set_error("rotary: pairs of an axis out of range"); return D2C_ERR_SHAPE; }
        pairs += p;
    }
    if (2 * pairs > q->D) { d2c_set_error("rotary: %ld pairs do not fit a head of %d channels", pairs, q->D); return D2C_ERR_SHAPE; }
    if (pairs > D2C_ROTARY_MAX_PAIRS) { d2c_set_error("rotary: up to %d pairs", D2C_ROTARY_MAX_PAIRS); return D2C_ERR_UNSUPPORTED; }
    if (q->direction != 1 && q->direction != -1) { d2c_set_error("rotary: direction must be 1 or -1"); return D2C_ERR_SHAPE; }
    if (!((float)q->base > 0.f) || !((float)q->base < INFINITY)) {      // (rates have to be floats)
        d2c_set_error("rotary: base must be positive and finite");
        return D2C_ERR_SHAPE;
    }
    return D2C_OK;
}

}  // namespace

extern "C" int d2c_rotary3d(const d2c_rotary3d_desc *q, const void *x, const float *positions, void *y, void *stream)
{
    if (int rc = check(q)) return rc;
    if (q->N == 0 || q->L == 0) return D2C_OK;
    if (!x || !y) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    if (!positions && (q->grid[0] <= 0 || q->grid[1] <= 0 || q->grid[2] <= 0 || (long)q->grid[0] * q->grid[1] * q->grid[2] != q->L)) {
        d2c_set_error("rotary: a grid of %d x %d x %d is not %d tokens", q->grid[0], q->grid[1], q->grid[2], q->L);
        return D2C_ERR_SHAPE;
    }
    RotArgs a{};
    a.x = x; a.pos = positions; a.y = y;
    for (int i = 0; i < 3; i++) a.xs[i] = q->x_stride[i];
    a.ps = q->position_stride;
    a.L = q->L; a.H = q->H; a.D = q->D;
    a.end0 = q->pairs[0]; a.end1 = a.end0 + q->pairs[1]; a.pairs = a.end1 + q->pairs[2];
    a.gh = std::max(q->grid[1], 1); a.gw = std::max(q->grid[2], 1);
    a.sign = (float)q->direction;
    int j = 0;
    for (int p : q->pairs)
        for (int i = 0; i < p; i++, j++) {
            const double rate = std::pow(q->base, -(double)i / p) * 0.15915494309189533577;
            a.hi[j] = (float)rate;
            a.lo[j] = (float)(rate - (double)a.hi[j]);
        }
    // Tokens to a workgroup: 16 KB of channels (more: cosines and sines wait longer for the first channels), fewer where that leaves compute units without one
    const long bytes = (long)q->H * q->D * (long)d2c_elem_size(q->dtype), fill = 4L * std::max(d2c_num_cus(), 1);
    long tokens = std::max(1L, std::min((16L << 10) / bytes, (long)q->N * q->L / fill));
    if (a.pairs > 0) tokens = std::min(tokens, (long)kRotLds / (a.pairs * 8L));
    a.tokens = (int)tokens;
    const dim3 grid((unsigned)((q->L + tokens - 1) / tokens), (unsigned)q->N);
    const size_t lds = (size_t)tokens * a.pairs * 8;
    hipStream_t st = (hipStream_t)stream;
    if (q->dtype == D2C_BF16) {
        if (q->interleaved) hipLaunchKernelGGL((rotary_kernel<bf16_t, true>), grid, dim3(kRotThreads), lds, st, a);
        else hipLaunchKernelGGL((rotary_kernel<bf16_t, false>), grid, dim3(kRotThreads), lds, st, a);
    } else {
        if (q->interleaved) hipLaunchKernelGGL((rotary_kernel<float, true>), grid, dim3(kRotThreads), lds, st, a);
        else hipLaunchKernelGGL((rotary_kernel<float, false>), grid, dim3(kRotThreads), lds, st, a);
    }
    return d2c_check_launch("rotary_kernel");
}
