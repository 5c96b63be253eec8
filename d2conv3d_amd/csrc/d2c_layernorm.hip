// Layer norm over the channels of a row, forward and backward.
//
//   mean = sum_c x / C,  var = sum_c (x - mean)^2 / C,  rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd,  y = xh w + b
//   grad_x = rstd (gw - A - xh B),   gw = grad_y w,  A = sum_c gw / C,  B = sum_c gw xh / C
//   grad_w = sum_rows grad_y xh,     grad_b = sum_rows grad_y
//
// Bound: memory.  LANES lanes hold a row in registers, NV 16-byte vectors each, so that x is read once and the variance is a sum of
// squared deviations from the mean itself.  Workgroups walk over the rows; in the backward pass each adds up its rows' part of grad_w and grad_b
// in registers on the way, and ln_params_kernel adds up the workgroups' sums, in their order.
#include <algorithm>
#include "d2c_common.hpp"
#include "d2c_mma.hpp"

namespace {

constexpr int kLnThreads = 256;

struct LnArgs {
    const void *x, *gy, *w, *b;
    void *y;                      // backward: grad_x (may be NULL)
    float *stats;                 // [rows][2]: mean, rstd
    float *part;                  // backward: [workgroups][2][C]
    void *gw, *gb;
    long rows, xs;
    int C, blocks;
    float eps;
};

// A lane's vectors of a row: NV pieces of 16 bytes, LANES pieces apart, zeros behind the row's end
template <typename T, int LANES, int NV> struct RowPart {
    static constexpr int VEC = 16 / (int)sizeof(T);
    uint4 v[NV];
    D2C_DEV void load(const T *row, int lane, int C)
    {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * LANES + lane) * VEC;
            v[i] = c < C ? load_run<T>(row + c, C - c) : make_uint4(0, 0, 0, 0);
        }
    }
    D2C_DEV void floats(int i, float *f) const
    {
        alignas(16) T e[VEC];
        *reinterpret_cast<uint4 *>(e) = v[i];
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] = elem_to_f32<T>(e[j]);
    }
};
// VEC parameters from channel c on (NULL: `none`)
template <typename TP, int VEC> D2C_DEV void load_params(const void *p, int c, int C, float none, float *f)
{
    constexpr int E = 16 / (int)sizeof(TP);
#pragma unroll
    for (int i = 0; i < VEC; i += E) {
        alignas(16) TP e[E];
        if (p && c + i < C) *reinterpret_cast<uint4 *>(e) = load_run<TP>(reinterpret_cast<const TP *>(p) + c + i, C - c - i);
        else {
#pragma unroll
            for (int j = 0; j < E; j++) e[j] = f32_to_elem<TP>(none);
        }
#pragma unroll
        for (int j = 0; j < E; j++) f[i + j] = elem_to_f32<TP>(e[j]);
    }
}

// Sum over the LANES lanes of a row
template <int LANES> D2C_DEV float row_sum(float v, float *red)
{
    v = lanes_sum<LANES < 64 ? LANES : 64>(v);
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0] + red[1] + red[2] + red[3];
    }
    return v;
}

// Rows are requested one ahead, and parameters stay in registers where they are few: what a wavefront has in flight while it sums bounds it (a row at a
// time, sums by shuffles, parameters read for each row, and so; us, bfloat16: 207360 rows of 256 52, 40.6 forward (5.2 TB/s), 61, 57 backward (5.6); 25920 of
// 512 15.4, 14.8 and 19.5, 18.0).
template <typename T, typename TP, int LANES, int NV> __global__ void __launch_bounds__(kLnThreads) ln_fwd_kernel(LnArgs a)
{
    constexpr int VEC = 16 / (int)sizeof(T), PER = kLnThreads / LANES;
    constexpr bool KEEP = NV * VEC <= 16;
    __shared__ float red[4];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float C = (float)a.C;
    const long step = (long)gridDim.x * PER;
    const T *xb = reinterpret_cast<const T *>(a.x);
    float w[KEEP ? NV : 1][VEC], b[KEEP ? NV : 1][VEC];
    RowPart<T, LANES, NV> next;
    long row = (long)blockIdx.x * PER + sub;
    next.load(xb + min(row, a.rows - 1) * a.xs, lane, a.C);
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            load_params<TP, VEC>(a.w, (i * LANES + lane) * VEC, a.C, 1.f, w[i]);
            load_params<TP, VEC>(a.b, (i * LANES + lane) * VEC, a.C, 0.f, b[i]);
        }
    }
    for (; row - sub < a.rows; row += step) {
        const RowPart<T, LANES, NV> now = next;
        if (row - sub + step < a.rows) next.load(xb + min(row + step, a.rows - 1) * a.xs, lane, a.C);
        float v[NV][VEC], s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            now.floats(i, v[i]);
#pragma unroll
            for (int j = 0; j < VEC; j++) s += v[i][j];
        }
        const float mean = row_sum<LANES>(s, red) / C;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * LANES + lane) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                v[i][j] = c + j < a.C ? v[i][j] - mean : 0.f;
                q = fmaf(v[i][j], v[i][j], q);
            }
        }
        const float rstd = 1.f / sqrtf(row_sum<LANES>(q, red) / C + a.eps);
        if (row >= a.rows) continue;
        T *y = reinterpret_cast<T *>(a.y) + row * a.C;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * LANES + lane) * VEC;
            if (c >= a.C) continue;
            if constexpr (!KEEP) {
                load_params<TP, VEC>(a.w, c, a.C, 1.f, w[0]);
                load_params<TP, VEC>(a.b, c, a.C, 0.f, b[0]);
            }
            alignas(16) T e[VEC];
#pragma unroll
            for (int j = 0; j < VEC; j++) e[j] = f32_to_elem<T>(fmaf(v[i][j] * rstd, w[KEEP ? i : 0][j], b[KEEP ? i : 0][j]));
            store_run<T>(y + c, *reinterpret_cast<const uint4 *>(e), a.C - c);
        }
        if (a.stats && lane == 0) *reinterpret_cast<float2 *>(a.stats + row * 2) = make_float2(mean, rstd);
    }
}

template <typename T, typename TP, int LANES, int NV> __global__ void __launch_bounds__(kLnThreads) ln_bwd_kernel(LnArgs a)
{
    constexpr int VEC = 16 / (int)sizeof(T), PER = kLnThreads / LANES;
    constexpr bool KEEP = NV * VEC <= 16;
    __shared__ float red[4];
    extern __shared__ float s_part[];      // [PER][C], where PER > 1
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float inv = 1.f / (float)a.C;
    const long step = (long)gridDim.x * PER;
    const T *xb = reinterpret_cast<const T *>(a.x), *gyb = reinterpret_cast<const T *>(a.gy);
    float gw[NV][VEC], gb[NV][VEC], w[KEEP ? NV : 1][VEC];
#pragma unroll
    for (int i = 0; i < NV; i++) {
#pragma unroll
        for (int j = 0; j < VEC; j++) gw[i][j] = gb[i][j] = 0.f;
        if constexpr (KEEP) load_params<TP, VEC>(a.w, (i * LANES + lane) * VEC, a.C, 1.f, w[i]);
    }
    RowPart<T, LANES, NV> nx, ng;
    float2 nst = make_float2(0.f, 0.f);
    auto request = [&](long row) INLINE {      // (rows behind the last repeat it: not added up, not stored)
        const long at = min(row, a.rows - 1);
        nx.load(xb + at * a.xs, lane, a.C);
        ng.load(gyb + at * a.C, lane, a.C);
        nst = *reinterpret_cast<const float2 *>(a.stats + at * 2);
    };
    long row = (long)blockIdx.x * PER + sub;
    if (row - sub < a.rows) request(row);
    for (; row - sub < a.rows; row += step) {
        const RowPart<T, LANES, NV> x = nx, g = ng;
        const float2 st = nst;
        const bool live = row < a.rows;
        if (row - sub + step < a.rows) request(row + step);
        float h[NV][VEC], t[NV][VEC], A = 0.f, B = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) x.floats(i, h[i]);
        if (!(fabsf(st.x * st.y) < INFINITY)) {      // (zeros behind a row's end would become infinities, and meet zeros)
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if ((i * LANES + lane) * VEC + j >= a.C) h[i][j] = st.x;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * LANES + lane) * VEC;
            g.floats(i, t[i]);
            if constexpr (!KEEP) load_params<TP, VEC>(a.w, c, a.C, 1.f, w[0]);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                h[i][j] = (h[i][j] - st.x) * st.y;
                if (!live) t[i][j] = 0.f;
                gw[i][j] = fmaf(t[i][j], h[i][j], gw[i][j]);
                gb[i][j] += t[i][j];
                t[i][j] *= w[KEEP ? i : 0][j];
                A += t[i][j];
                B = fmaf(t[i][j], h[i][j], B);
            }
        }
        if (!a.y) continue;
        A = row_sum<LANES>(A, red) * inv;
        B = row_sum<LANES>(B, red) * inv;
        if (!live) continue;
        T *y = reinterpret_cast<T *>(a.y) + row * a.C;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * LANES + lane) * VEC;
            if (c >= a.C) continue;
            alignas(16) T e[VEC];
#pragma unroll
            for (int j = 0; j < VEC; j++) e[j] = f32_to_elem<T>(st.y * (t[i][j] - A - h[i][j] * B));
            store_run<T>(y + c, *reinterpret_cast<const uint4 *>(e), a.C - c);
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float *out = a.part + ((long)blockIdx.x * 2 + which) * a.C;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const int c = (i * LANES + lane) * VEC + j;
                if (c >= a.C) continue;
                const float v = which ? gb[i][j] : gw[i][j];
                if constexpr (PER > 1) s_part[sub * a.C + c] = v;
                else out[c] = v;
            }
        if constexpr (PER > 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < a.C; c += kLnThreads) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < PER; k++) v += s_part[k * a.C + c];
                out[c] = v;
            }
        }
    }
}

// The workgroups' sums: 64 channels (16 lanes of four) and 64 slices of the workgroups to a workgroup here.  Bound: latency, a slice's few loads are in flight
// together (16 slices of 64 loads each, 1024 workgroups: 20 us).
constexpr int kLnSlices = 64;
template <typename TP> __global__ void __launch_bounds__(16 * kLnSlices) ln_params_kernel(LnArgs a)
{
    __shared__ float4 s[kLnSlices][16];
    const int lane = threadIdx.x & 15, c = (int)blockIdx.x * 64 + lane * 4, slice = threadIdx.x >> 4, which = blockIdx.y;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C) {
#pragma unroll 8
        for (int k = slice; k < a.blocks; k += kLnSlices) {
            const float4 p = __builtin_bit_cast(float4, load_run<float>(a.part + ((long)k * 2 + which) * a.C + c, a.C - c));
            v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w;
        }
    }
    s[slice][lane] = make_float4(v[0], v[1], v[2], v[3]);
#pragma unroll
    for (int n = kLnSlices / 2; n > 0; n >>= 1) {
        __syncthreads();
        if (slice < n) {
            const float4 p = s[slice][lane], q = s[slice + n][lane];
            s[slice][lane] = make_float4(p.x + q.x, p.y + q.y, p.z + q.z, p.w + q.w);
        }
    }
    if (slice != 0 || c >= a.C) return;
    const float4 p = s[0][lane];
    const float r[4] = {p.x, p.y, p.z, p.w};
    TP *out = reinterpret_cast<TP *>(which ? a.gb : a.gw);
    if (!out) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (c + i < a.C) out[c + i] = f32_to_elem<TP>(r[i]);
}

constexpr int kLnMaxChannels = 16384;

int check(const d2c_layer_norm_desc *q)
{
    if (!q) { d2c_set_error("layer norm: null description"); return D2C_ERR_SHAPE; }
    if (q->rows < 0 || q->C <= 0) { d2c_set_error("layer norm: rows must not be negative, channels positive"); return D2C_ERR_SHAPE; }
    if (q->dtype != D2C_F32 && q->dtype != D2C_BF16) { d2c_set_error("layer norm: float32 or bfloat16 only"); return D2C_ERR_DTYPE; }
    if (q->param_dtype != q->dtype && q->param_dtype != D2C_F32) { d2c_set_error("layer norm: parameters of the input's type or float32"); return D2C_ERR_DTYPE; }
    if (q->C > kLnMaxChannels) { d2c_set_error("layer norm: up to %d channels, got %d", kLnMaxChannels, q->C); return D2C_ERR_UNSUPPORTED; }
    if (!(q->eps >= 0.f)) { d2c_set_error("layer norm: eps must be non-negative"); return D2C_ERR_SHAPE; }
    return D2C_OK;
}

// Lanes to a row and vectors to a lane: one vector as long as a row fits a wavefront's lanes, then up to four, then a workgroup to a row
struct LnShape { int lanes, nv; };
LnShape shape_of(const d2c_layer_norm_desc &q)
{
    const int vec = q.dtype == D2C_BF16 ? 8 : 4, n = (q.C + vec - 1) / vec;
    for (int lanes : {8, 16, 32, 64})
        if (n <= lanes) return {lanes, 1};
    if (n <= 128) return {64, 2};
    if (n <= 256) return {64, 4};
    if (n <= 1024) return {256, 4};
    return {256, 16};
}
// `most`: no more than so many (backward: workgroups' sums of up to 64 MB)
constexpr long kLnPartBytes = 64L << 20;
long most_blocks(const d2c_layer_norm_desc &q) { return kLnPartBytes / (2L * q.C * (long)sizeof(float)); }
int blocks_of(const d2c_layer_norm_desc &q, const LnShape &s, int per_cu, long most = 1L << 30)
{
    const long per = kLnThreads / s.lanes;
    return (int)std::max(1L, std::min((q.rows + per - 1) / per, std::min((long)per_cu * std::max(d2c_num_cus(), 1), most)));
}
constexpr int kFwdPerCu = 16, kBwdPerCu = 4;      // (8 and 16: 43.8, 40.6 us forward on 207360 rows of 256; 2, 4, 8: 66, 57, 61 us backward)

template <bool BWD, typename T, typename TP, int LANES, int NV> int launch_shape(const LnArgs &a, hipStream_t st)
{
    if constexpr (BWD) {
        const int lds = LANES < 256 && a.part ? kLnThreads / LANES * a.C * 4 : 0;
        hipLaunchKernelGGL((ln_bwd_kernel<T, TP, LANES, NV>), dim3((unsigned)a.blocks), dim3(kLnThreads), lds, st, a);
        return d2c_check_launch("ln_bwd_kernel");
    } else {
        hipLaunchKernelGGL((ln_fwd_kernel<T, TP, LANES, NV>), dim3((unsigned)a.blocks), dim3(kLnThreads), 0, st, a);
        return d2c_check_launch("ln_fwd_kernel");
    }
}
template <bool BWD, typename T, typename TP> int launch_types(const LnArgs &a, const LnShape &s, hipStream_t st)
{
    switch (s.lanes * 100 + s.nv) {
    case 801: return launch_shape<BWD, T, TP, 8, 1>(a, st);
    case 1601: return launch_shape<BWD, T, TP, 16, 1>(a, st);
    case 3201: return launch_shape<BWD, T, TP, 32, 1>(a, st);
    case 6401: return launch_shape<BWD, T, TP, 64, 1>(a, st);
    case 6402: return launch_shape<BWD, T, TP, 64, 2>(a, st);
    case 6404: return launch_shape<BWD, T, TP, 64, 4>(a, st);
    case 25604: return launch_shape<BWD, T, TP, 256, 4>(a, st);
    default: return launch_shape<BWD, T, TP, 256, sizeof(T) == 2 ? 8 : 16>(a, st);
    }
}
template <bool BWD> int launch(const d2c_layer_norm_desc &q, const LnArgs &a, const LnShape &s, hipStream_t st)
{
    if (q.dtype == D2C_F32) return launch_types<BWD, float, float>(a, s, st);
    if (q.param_dtype == D2C_F32) return launch_types<BWD, bf16_t, float>(a, s, st);
    return launch_types<BWD, bf16_t, bf16_t>(a, s, st);
}

}  // namespace

extern "C" int d2c_layer_norm_forward(const d2c_layer_norm_desc *q, const void *x, const void *weight, const void *bias, void *y,
                                      float *stats, void *stream)
{
    if (int rc = check(q)) return rc;
    if (q->rows == 0) return D2C_OK;
    if (!x || !y) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    const LnShape s = shape_of(*q);
    const LnArgs a{x, nullptr, weight, bias, y, stats, nullptr, nullptr, nullptr, q->rows, q->x_stride, q->C, blocks_of(*q, s, kFwdPerCu), q->eps};
    return launch<false>(*q, a, s, (hipStream_t)stream);
}

extern "C" size_t d2c_layer_norm_backward_workspace_bytes(const d2c_layer_norm_desc *q)
{
    if (check(q) != D2C_OK) return 0;
    return d2c_align_up((size_t)blocks_of(*q, shape_of(*q), kBwdPerCu, most_blocks(*q)) * 2 * q->C * sizeof(float));
}

extern "C" int d2c_layer_norm_backward(const d2c_layer_norm_desc *q, const void *grad_y, const void *x, const float *stats,
                                       const void *weight, void *grad_x, void *grad_weight, void *grad_bias, void *ws,
                                       size_t ws_bytes, void *stream)
{
    if (int rc = check(q)) return rc;
    if (q->rows > 0 && (!grad_y || !x || !stats)) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    const bool params = grad_weight || grad_bias;
    const size_t need = d2c_layer_norm_backward_workspace_bytes(q);
    if (params && (!ws || ws_bytes < need || ((uintptr_t)ws & 255u))) {
        d2c_set_error("workspace of %zu bytes (256-byte aligned) required, got %zu at %p", need, ws_bytes, ws);
        return D2C_ERR_WORKSPACE;
    }
    const LnShape s = shape_of(*q);
    const LnArgs a{x, grad_y, weight, nullptr, grad_x, const_cast<float *>(stats), params ? (float *)ws : nullptr, grad_weight, grad_bias, q->rows,
                   q->x_stride, q->C, blocks_of(*q, s, kBwdPerCu, most_blocks(*q)), q->eps};
    hipStream_t st = (hipStream_t)stream;
    if (q->rows > 0 || params)
        if (int rc = launch<true>(*q, a, s, st)) return rc;      // (no rows: sums of nothing)
    if (!params) return D2C_OK;
    const dim3 grid((unsigned)((q->C + 63) / 64), 2);
    if (q->param_dtype == D2C_F32) hipLaunchKernelGGL(ln_params_kernel<float>, grid, dim3(16 * kLnSlices), 0, st, a);
    else hipLaunchKernelGGL(ln_params_kernel<bf16_t>, grid, dim3(16 * kLnSlices), 0, st, a);
    return d2c_check_launch("ln_params_kernel");
}
