// Attention of one map's positions to those of another: forward pass.  Formulas and operand orders: d2c_attention.hpp.
//
// A workgroup takes one key head, 128 rows (32 to a wavefront) and walks over the keys a tile at a time, K and V through LDS, the
// next tile requested while this one is worked on.  Few rows: the wavefronts share them and split the keys of a tile, and several workgroups share the keys;
// their results are joined by attn_join_kernel.
#include <algorithm>
#include "d2c_attention.hpp"

using namespace d2c_attn;

namespace {

// The keys of a tile that are to be read: bit i of word j is key k0 + 64 j + i.  Requested as bytes two tiles ahead.
template <int WORDS> struct KeyBits {
    bool b[WORDS];
    D2C_DEV void request(const Args &a, int n, int keys, int k0)
    {
#pragma unroll
        for (int j = 0; j < WORDS; j++) {
            const int key = k0 + j * 64 + (int)(threadIdx.x & 63);
            b[j] = key < keys && (!a.mask || a.mask[(long)n * a.Lk + key]);
        }
    }
    D2C_DEV void words(uint64_t (&w)[WORDS]) const
    {
#pragma unroll
        for (int j = 0; j < WORDS; j++) w[j] = __ballot(b[j]);
    }
};

template <typename T, int DP, int WK, bool WHOLE> struct FwdShape {
    static constexpr int KW = sizeof(T) == 2 && WK == 1 ? 64 : 32, KT = KW * WK, ROWS = 32 * (4 / WK);
    using KV = Tile<T, DP, KT, 256, WHOLE>;
    static constexpr int JOIN = WK > 1 ? 4 * 32 * (DP + 2) * 4 : 0;
    static constexpr int LDS = 2 * KV::BYTES > JOIN ? 2 * KV::BYTES : JOIN;
};

// WK: wavefronts that share rows and split the keys of a tile
template <typename T, int DP, int WK, bool WHOLE> __global__ void __launch_bounds__(256, 2) attn_fwd_kernel(Args a)
{
    using Shape = FwdShape<T, DP, WK, WHOLE>;
    using KV = typename Shape::KV;
    constexpr int P = kTerms<T>, NK = DP / 16, ND = DP / 32, KW = Shape::KW, KT = Shape::KT, NS = KW / 32, WORDS = (KT + 63) / 64;
    extern __shared__ __align__(16) unsigned char lds[];
    unsigned char *s_k = lds, *s_v = lds + KV::BYTES;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, wk = wave % WK;
    const Head hd = head_of(a);
    const int row = (int)blockIdx.y * Shape::ROWS + (wave / WK) * 32 + (lane & 31);
    const int keys = keys_of(a, hd.n), tiles = (keys + KT - 1) / KT;
    const int split = (int)blockIdx.z, t1 = (int)((long)tiles * (split + 1) / a.splits);
    int t = (int)((long)tiles * split / a.splits);

    const T *kb = reinterpret_cast<const T *>(a.k) + hd.n * a.ks[0] + hd.h * a.ks[2];
    const T *vb = reinterpret_cast<const T *>(a.v) + hd.n * a.vs[0] + hd.h * a.vs[2];
    KV k, v;
    KeyBits<WORDS> bits;
    uint64_t next[WORDS];
    auto request = [&](int tile) INLINE {
        const int any = any_key(next);
        if (any < 0) return;
        const T *kt = kb + (long)tile * KT * a.ks[1], *vt = vb + (long)tile * KT * a.vs[1];
        k.load(a.D, [&](int i) INLINE { return kt + key_to_load(next, i, any) * a.ks[1]; });
        v.load(a.D, [&](int i) INLINE { return vt + key_to_load(next, i, any) * a.vs[1]; });
    };
    if (t < t1) {
        bits.request(a, hd.n, keys, t * KT);
        bits.words(next);
        request(t);
        bits.request(a, hd.n, keys, (t + 1) * KT);
    }
    Frag<P> q[NK];
    {
        const T *qr = row_at<T>(a.q, a.qs, a, hd, min(row, a.rows - 1));
#pragma unroll
        for (int i = 0; i < NK; i++) {
            const int d = i * 16 + half * 8;
            q[i] = terms_of<T>(load8_of<WHOLE, T>(qr, d, a.D, row < a.rows));
        }
    }
    f32x16 o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[i][r] = 0.f;
    float m = -INFINITY, lift = -INFINITY, l = 0.f;
    const float c = a.scale2;

    for (; t < t1; t++) {
        uint64_t now[WORDS];
#pragma unroll
        for (int j = 0; j < WORDS; j++) now[j] = next[j];
        __syncthreads();
        k.store(s_k);
        v.store(s_v);
        __syncthreads();
        if (t + 1 < t1) {
            bits.words(next);
            request(t + 1);
            bits.request(a, hd.n, keys, (t + 2) * KT);
        }
        const uint64_t mine = now[wk * KW / 64] >> (wk * KW % 64);
        if ((KW == 64 ? mine : (mine & 0xffffffffu)) == 0) continue;
        f32x16 s[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[i][r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NK; ks++) mma<P>(s[i], KV::rows(s_k, wk * KW + i * 32 + (lane & 31), ks, half), q[ks]);
            const uint32_t there = (uint32_t)(mine >> (i * 32));
            if (there != 0xffffffffu) {
                const uint32_t b = there >> (half * 4);
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!((b >> (8 * (r / 4) + r % 4)) & 1)) s[i][r] = -INFINITY;
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[i][r]);
        // (a row's maximum follows only where it has grown by a factor of 2^8 of the weights: what is added up stays far from float32's
        // ends, and the sums are seldom scaled anew)
        if (__any(top > lift)) {
            const float grown = half_max(top);
            if (grown > lift) {
                const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - grown) * c);
                m = grown;
                lift = m + 8.f / c;
                l *= f;
#pragma unroll
                for (int i = 0; i < ND; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[i][r] *= f;
            }
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            float p[16];
#pragma unroll
            for (int r = 0; r < 16; r++) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], c, -mc));
                l += p[r];
            }
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                const Frag<P> pf = make_frag<P>(p + kk * 8);
#pragma unroll
                for (int d = 0; d < ND; d++) mma<P>(o[d], KV::columns(s_v, wk * KW + i * 32 + kk * 16, d * 32, lane), pf);
            }
        }
    }
    l = half_sum(l);
    float mc = m == -INFINITY ? -INFINITY : m * c;

    if constexpr (WK > 1) {
        // the wavefronts of the same rows: sums through LDS, [wavefront][lane of 32][DP], then (mc, l)
        float *s_o = reinterpret_cast<float *>(lds), *s_ml = s_o + 4 * 32 * DP;
        __syncthreads();
        if (half == 0) { s_ml[(wave * 32 + lane) * 2] = mc; s_ml[(wave * 32 + lane) * 2 + 1] = l; }
        __syncthreads();
        const int first = wave / WK * WK;
        float all = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; w++) all = fmaxf(all, s_ml[((first + w) * 32 + (lane & 31)) * 2]);
        const float base = all == -INFINITY ? 0.f : all;
#pragma unroll
        for (int w = 0; w < WK; w++)
            sum += s_ml[((first + w) * 32 + (lane & 31)) * 2 + 1] * __builtin_amdgcn_exp2f(s_ml[((first + w) * 32 + (lane & 31)) * 2] - base);
        const float f = __builtin_amdgcn_exp2f(mc - base);
        // (a lane's values: its row's columns 32 i + 8 j + 4 half ..)
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) s_o[(wave * DP + i * 32 + 8 * (r / 4) + 4 * half + r % 4) * 32 + (lane & 31)] = o[i][r] * f;
        __syncthreads();
        if (wk != 0) return;
        mc = all; l = sum;
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < WK; w++) x += s_o[((first + w) * DP + i * 32 + 8 * (r / 4) + 4 * half + r % 4) * 32 + (lane & 31)];
                o[i][r] = x;
            }
    }
    if (row >= a.rows) return;
    if (a.splits > 1) {
        const long at = ((long)split * gridDim.x + hd.nh) * a.rows + row;
        float *po = a.part + at * a.D;
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int d = i * 32 + j * 8 + half * 4;
                const float x[4] = {o[i][j * 4], o[i][j * 4 + 1], o[i][j * 4 + 2], o[i][j * 4 + 3]};
                store4<float>(po + d, x, a.D - d);
            }
        if (half == 0) { a.part_ml[at * 2] = mc; a.part_ml[at * 2 + 1] = l; }
        return;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // (no key: 0; a sum that is NaN stays one)
    const int pos = row / a.group, head = hd.h * a.group + row - pos * a.group;
    T *orow = reinterpret_cast<T *>(a.out) + (((long)hd.n * a.Lq + pos) * a.Hq + head) * a.D;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + j * 8 + half * 4;
            const float x[4] = {o[i][j * 4] * inv, o[i][j * 4 + 1] * inv, o[i][j * 4 + 2] * inv, o[i][j * 4 + 3] * inv};
            store4<T>(orow + d, x, a.D - d);
        }
    if (a.lse && half == 0) a.lse[hd.nh * a.rows + row] = l == 0.f ? INFINITY : mc + log2f(l);
}

// The partial results of `splits` workgroups.  LANES lanes take four of a row's columns each, `groups` (a power of two) of them the splits in turn; their sums
// meet in LDS.  Latency counts: one row of 102 splits 13.6 us as a wavefront that walks over them, JOIN_FEW as here.
template <typename T, int LANES> __global__ void __launch_bounds__(256) attn_join_kernel(Args a, int groups)
{
    __shared__ float4 s_x[256];
    __shared__ float2 s_ml[256];
    const int per = 256 / (LANES * groups), lane = threadIdx.x % LANES, group = threadIdx.x / LANES % groups;
    const long total = (long)a.N * a.Hkv * a.rows, at = (long)blockIdx.x * per + threadIdx.x / (LANES * groups);
    const bool live = at < total;
    const int d = lane * 4;
    float all = -INFINITY, l = 0.f;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
#pragma unroll 4
        for (int s = group; s < a.splits; s += groups) {
            const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + (s * total + at) * 2);
            const float4 y = __builtin_bit_cast(float4, d < a.D ? load_run<float>(a.part + (s * total + at) * a.D + d, a.D - d) : make_uint4(0, 0, 0, 0));
            const float top = fmaxf(all, ml.x), base = top == -INFINITY ? 0.f : top;
            const float f = __builtin_amdgcn_exp2f(all - base), g = __builtin_amdgcn_exp2f(ml.x - base);
            all = top;
            l = l * f + ml.y * g;
            x[0] = x[0] * f + y.x * g; x[1] = x[1] * f + y.y * g; x[2] = x[2] * f + y.z * g; x[3] = x[3] * f + y.w * g;
        }
    }
    s_x[threadIdx.x] = make_float4(x[0], x[1], x[2], x[3]);
    s_ml[threadIdx.x] = make_float2(all, l);
    __syncthreads();
    if (group != 0 || !live) return;
    float top = all;
    for (int g = 1; g < groups; g++) top = fmaxf(top, s_ml[threadIdx.x + g * LANES].x);
    const float base = top == -INFINITY ? 0.f : top;
    l = x[0] = x[1] = x[2] = x[3] = 0.f;
    for (int g = 0; g < groups; g++) {
        const float2 ml = s_ml[threadIdx.x + g * LANES];
        const float4 y = s_x[threadIdx.x + g * LANES];
        const float f = __builtin_amdgcn_exp2f(ml.x - base);
        l = fmaf(ml.y, f, l);
        x[0] = fmaf(y.x, f, x[0]); x[1] = fmaf(y.y, f, x[1]); x[2] = fmaf(y.z, f, x[2]); x[3] = fmaf(y.w, f, x[3]);
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const long nh = at / a.rows;
    const int row = (int)(at - nh * a.rows), n = (int)(nh / a.Hkv), pos = row / a.group;
    const int head = (int)(nh - (long)n * a.Hkv) * a.group + row - pos * a.group;
    T *orow = reinterpret_cast<T *>(a.out) + (((long)n * a.Lq + pos) * a.Hq + head) * a.D;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] *= inv;
    if (d < a.D) store4<T>(orow + d, x, a.D - d);
    if (a.lse && lane == 0) a.lse[at] = l == 0.f ? INFINITY : top + log2f(l);
}

// What a call runs on: rows of 32 or fewer are shared by the wavefronts of a workgroup (WK > 1), and so many workgroups share the keys that there
// are two to a compute unit, each with a tile at least.
struct FwdPlan { int wk, row_tiles, splits; size_t part_bytes, bytes; };
FwdPlan fwd_plan(const d2c_attention_desc &q)
{
    FwdPlan p;
    const long rows = (long)q.Lq * (q.Hq / q.Hkv), heads = (long)q.N * q.Hkv;
    const bool bf = q.dtype == D2C_BF16;
    p.wk = rows <= 32 ? (bf ? 4 : 2) : 1;
    const int tile_rows = 32 * (4 / p.wk), tile_keys = p.wk > 1 ? 32 * p.wk : (bf ? 64 : 32);
    p.row_tiles = (int)((rows + tile_rows - 1) / tile_rows);
    const long groups = std::max(heads * p.row_tiles, 1L), tiles = (q.Lk + tile_keys - 1) / tile_keys;
    p.splits = (int)std::max(1L, std::min(2L * std::max(d2c_num_cus(), 1) / groups, tiles));
    p.part_bytes = p.splits > 1 ? d2c_align_up((size_t)p.splits * heads * rows * q.D * 4) : 0;
    p.bytes = p.splits > 1 ? p.part_bytes + d2c_align_up((size_t)p.splits * heads * rows * 8) : 0;
    return p;
}

template <typename T, int DP, int WK, bool WHOLE> int launch_fwd(const Args &a, const FwdPlan &p, hipStream_t st)
{
    constexpr int lds = FwdShape<T, DP, WK, WHOLE>::LDS;
    const void *kernel = reinterpret_cast<const void *>(&attn_fwd_kernel<T, DP, WK, WHOLE>);
    if (int rc = d2c_allow_lds(kernel, lds, "attn_fwd_kernel")) return rc;
    hipLaunchKernelGGL((attn_fwd_kernel<T, DP, WK, WHOLE>), dim3((unsigned)(a.N * a.Hkv), (unsigned)p.row_tiles, (unsigned)p.splits), dim3(256), lds, st, a);
    return d2c_check_launch("attn_fwd_kernel");
}
template <typename T, int DP> int launch_fwd_d(const Args &a, const FwdPlan &p, hipStream_t st)
{
    constexpr int WK = sizeof(T) == 2 ? 4 : 2;
    if (a.D % 8 == 0) return p.wk > 1 ? launch_fwd<T, DP, WK, true>(a, p, st) : launch_fwd<T, DP, 1, true>(a, p, st);
    return p.wk > 1 ? launch_fwd<T, DP, WK, false>(a, p, st) : launch_fwd<T, DP, 1, false>(a, p, st);
}
template <typename T, int LANES> int launch_join(const Args &a, hipStream_t st)
{
    int groups = 1;
    while (groups * 2 <= std::min(a.splits, 256 / LANES)) groups *= 2;
    const long total = (long)a.N * a.Hkv * a.rows, per = 256 / (LANES * groups);
    hipLaunchKernelGGL((attn_join_kernel<T, LANES>), dim3((unsigned)((total + per - 1) / per)), dim3(256), 0, st, a, groups);
    return d2c_check_launch("attn_join_kernel");
}
template <typename T> int launch_fwd_t(const Args &a, const FwdPlan &p, hipStream_t st)
{
    int rc;
    if (a.D <= 32) rc = launch_fwd_d<T, 32>(a, p, st);
    else if (a.D <= 64) rc = launch_fwd_d<T, 64>(a, p, st);
    else if (a.D <= 96) rc = launch_fwd_d<T, 96>(a, p, st);
    else rc = launch_fwd_d<T, 128>(a, p, st);
    if (rc || p.splits == 1) return rc;
    if (a.D <= 32) return launch_join<T, 8>(a, st);
    if (a.D <= 64) return launch_join<T, 16>(a, st);
    return launch_join<T, 32>(a, st);
}

}  // namespace

int d2c_attention_check(const d2c_attention_desc *q)
{
    if (!q) { d2c_set_error("attention: null description"); return D2C_ERR_SHAPE; }
    if (q->dtype != D2C_F32 && q->dtype != D2C_BF16) { d2c_set_error("attention: float32 or bfloat16 only"); return D2C_ERR_DTYPE; }
    if (q->N < 0 || q->Lq < 0 || q->Lk < 0 || q->Hq <= 0 || q->Hkv <= 0 || q->D <= 0) {
        d2c_set_error("attention: sizes must not be negative, heads and their size positive");
        return D2C_ERR_SHAPE;
    }
    if (q->Hq % q->Hkv != 0) { d2c_set_error("attention: %d query heads are no multiple of %d key heads", q->Hq, q->Hkv); return D2C_ERR_SHAPE; }
    if (q->D > 128) { d2c_set_error("attention: heads of up to 128 channels, got %d", q->D); return D2C_ERR_UNSUPPORTED; }
    if (!(q->scale > 0.f) || !(q->scale < INFINITY)) { d2c_set_error("attention: scale must be positive and finite"); return D2C_ERR_SHAPE; }
    // (a launch's second and third dimension end at 65535)
    if ((long)q->N * q->Hkv >= (1L << 31) || (long)q->Lq * (q->Hq / q->Hkv) > 65535L * 32 || q->Lk > 65535 * 32) {
        d2c_set_error("attention: too many samples, positions or heads");
        return D2C_ERR_SHAPE;
    }
    return D2C_OK;
}

Args d2c_attn::make_args(const d2c_attention_desc &q)
{
    Args a{};
    for (int i = 0; i < 3; i++) { a.qs[i] = q.q_stride[i]; a.ks[i] = q.k_stride[i]; a.vs[i] = q.v_stride[i]; }
    a.N = q.N; a.Lq = q.Lq; a.Lk = q.Lk; a.Hq = q.Hq; a.Hkv = q.Hkv; a.group = q.Hq / q.Hkv; a.D = q.D;
    a.rows = a.Lq * a.group;
    a.gs[0] = (long)q.Lq * q.Hq * q.D; a.gs[1] = (long)q.Hq * q.D; a.gs[2] = q.D;
    a.scale = q.scale; a.scale2 = q.scale * 1.44269504088896340736f;
    a.splits = 1;
    return a;
}

extern "C" size_t d2c_attention_forward_workspace_bytes(const d2c_attention_desc *q)
{
    return d2c_attention_check(q) == D2C_OK ? fwd_plan(*q).bytes : 0;
}

extern "C" int d2c_attention_forward(const d2c_attention_desc *q, const void *query, const void *key, const void *value,
                                     const int32_t *key_lengths, const uint8_t *key_mask, void *out, float *lse, void *ws,
                                     size_t ws_bytes, void *stream)
{
    if (int rc = d2c_attention_check(q)) return rc;
    if (q->N == 0 || q->Lq == 0) return D2C_OK;
    if (!query || !out || (q->Lk > 0 && (!key || !value))) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    const FwdPlan p = fwd_plan(*q);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 255u))) {
        d2c_set_error("workspace of %zu bytes (256-byte aligned) required, got %zu at %p", p.bytes, ws_bytes, ws);
        return D2C_ERR_WORKSPACE;
    }
    Args a = make_args(*q);
    a.q = query; a.k = key; a.v = value; a.lengths = key_lengths; a.mask = key_mask; a.out = out; a.lse = lse;
    a.splits = p.splits;
    a.part = (float *)ws; a.part_ml = (float *)((char *)ws + p.part_bytes);
    return q->dtype == D2C_BF16 ? launch_fwd_t<bf16_t>(a, p, (hipStream_t)stream) : launch_fwd_t<float>(a, p, (hipStream_t)stream);
}
