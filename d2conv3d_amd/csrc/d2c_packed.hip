// Attention inside sequences that lie behind each other: forward pass.  Shared parts: d2c_packed.hpp.
//
// A workgroup takes one key head and 128 rows of one sequence (32 to a wavefront) and walks over the keys that the last of them reads, a tile at a time, K and V
// through LDS, the next tile requested while this one is worked on.
#include "d2c_packed.hpp"

using namespace d2c_packed;

namespace {

template <typename T, int DP, bool WHOLE> struct FwdShape {
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;
    using KV = Tile<T, DP, KT, 256, WHOLE>;
    static constexpr int BUFFERS = 4 * KV::BYTES <= 52 << 10 ? 2 : 1;
    static constexpr int LDS = 2 * BUFFERS * KV::BYTES;
    // to a SIMD (said, the compiler uses 163 registers at 64 channels, of the 168 that three have; else 152: one sequence of 25920, 8 heads of 64, 0.82 ms, 0.84)
    static constexpr int WAVES = sizeof(T) == 2 && DP <= 64 ? 3 : 2;
};

// One pass over the keys with the running maximum and sum of a softmax, as attn_fwd_kernel; the weights go from one product's accumulator into the next one's operand in registers.
// Only tiles in which some row has a key that it does not read look at limits, and clean the values that others read from infinities and NaN (take_in brings them back).  Registers: what three
// workgroups of a compute unit have room for at 64 channels.  Bound: matrix instructions and the exponentials, maxima, sums and roundings between them.
// Measured, bfloat16: 16 pieces of up to 4096 queries on up to 12288 keys, 16 heads of 128 that share 4, 1.93 ms (0.97 PFLOP/s; a library product of 8192 cubed 1.22); one sequence of 25920, 8
// heads of 64 that share 2, 0.80 ms (0.86); six of up to 12960 in frames of 1620, 8 heads of 64, 0.73 ms (0.79).  float32: three of up to 1417, 6 heads of 40, 32 us and the join 5.1.
template <typename T, int DP, int NP, bool WHOLE, int PW> D2C_DEV void fwd_rows(const PackedArgs &a, const PackedUnit &u)
{
    using Shape = FwdShape<T, DP, WHOLE>;
    using KV = typename Shape::KV;
    constexpr int P = kTerms<T>, ND = DP / 32, NK = kSteps<NP>, KT = Shape::KT, NS = KT / 32, BUFFERS = Shape::BUFFERS;
    constexpr bool END = WHOLE && NP % 2 == 1;
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ int s_bad;      // whether a tile's values were cleaned
    if (threadIdx.x == 0) s_bad = 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, row0 = u.tile * kRows;
    const int tile_row = wave * 32 + (lane & 31), row = row0 + tile_row;
    const bool live = row < u.rows;
    // limits rise with the rows: this lane's, the smallest of the workgroup's, the largest and the smallest of the wavefront's
    const int lim = live ? limit_of_row(a, u, row) : 0, least = limit_of_row(a, u, row0);
    const int wave_row = row0 + wave * 32, wave_least = wave_row < u.rows ? limit_of_row(a, u, wave_row) : 0;
    const int wave_most = wave_row < u.rows ? limit_of_row(a, u, min(wave_row + 31, u.rows - 1)) : 0;
    const Walk walk = row_walk(a, u);
    if (u.split >= walk.splits) return;
    const int t1 = (int)((long)walk.steps * (u.split + 1) / walk.splits);
    const int t0 = (int)((long)walk.steps * u.split / walk.splits);
    int t = t0;

    KV k, v;
    const PackedKeyTiles<T, KV, KT, WHOLE> source(a, u);
    if (t < t1) source.request(a, k, v, t, u.lk - t * KT);
    Frag<P> q[NK];
    {
        const T *qr = row_at<T>(a.q, a.qs, a, u, min(row, u.rows - 1));
#pragma unroll
        for (int i = 0; i < NK; i++) {
            const int d = i * 16 + half * 8;
            const Raw8<T> raw = load8_of<WHOLE, T>(qr, d, a.D, live);
            if constexpr (sizeof(T) == 2) q[i] = terms_of<T>(raw);
            else {
                float x[8];
                floats_of<T>(raw, x);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] *= a.scale2;
                q[i] = make_frag<3, READ>(x);
            }
        }
    }
    f32x16 o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[i][r] = 0.f;
    float m = -INFINITY, lift = -INFINITY, l = 0.f;
    const float c = sizeof(T) == 4 ? 1.f : a.scale2;      // (float32 has its scale in the rows already)
    int buffer = 0;
    __syncthreads();

    for (; t < t1; t++) {
        unsigned char *s_k = lds + (BUFFERS == 2 ? buffer * 2 * KV::BYTES : 0), *s_v = s_k + KV::BYTES;
        const bool masked = t * KT + KT > least;
        if constexpr (BUFFERS == 1) __syncthreads();
        if (masked) {
            const int left = u.lk - t * KT;
            v.zero_rows([&](int i) INLINE { return i >= left; });      // (an infinite value that is repeated behind the sequence's end)
            if (__any(not_finite<T>(v))) {
                clean<T>(v);
                if (lane == 0) s_bad = 1;
            }
        }
        k.template store<END>(s_k, a.D);
        v.template store<false>(s_v, a.D);
        __syncthreads();
        if (t + 1 < t1) source.request(a, k, v, t + 1, u.lk - (t + 1) * KT);
        buffer ^= 1;
        if (t * KT >= wave_most) continue;
        f32x16 s[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[i][r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NK; ks++) mma(s[i], KV::rows(s_k, i * 32 + (lane & 31), ks, half), q[ks]);
            if (t * KT + i * 32 + 32 > wave_least) {
                const int left = lim - (t * KT + i * 32 + half * 4);
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (8 * (r / 4) + r % 4 >= left) s[i][r] = -INFINITY;
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[i][r]);
        // (a row's maximum follows only where it has grown by a factor of 2^8 of the weights)
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
                const Frag<PW> pf = make_frag<PW, WEIGHTS>(p + kk * 8);
#pragma unroll
                for (int d = 0; d < ND; d++) mma(o[d], KV::columns(s_v, i * 32 + kk * 16, d * 32, lane), pf);
            }
        }
    }
    __syncthreads();
    if (s_bad)
        take_in<T, false>(o, a.D, max(least / KT, t0) * KT, min(t1 * KT, wave_most), [&](int j) INLINE { return source.vb + (long)j * source.vs; },
                          [&](int j) INLINE { return j < lim; });
    l = half_sum(l);
    const float mc = m == -INFINITY ? -INFINITY : m * c;
    if (!live) return;
    if (walk.splits > 1) {
        const long at = (((long)u.split * a.tiles + u.at) * a.Hkv + u.h) * kRows + tile_row;
        float *po = a.part + at * part_width(a.D);
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
    T *orow = const_cast<T *>(row_at<T>(a.out, a.gs, a, u, row));
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + j * 8 + half * 4;
            const float x[4] = {o[i][j * 4] * inv, o[i][j * 4 + 1] * inv, o[i][j * 4 + 2] * inv, o[i][j * 4 + 3] * inv};
            store4<T>(orow + d, x, a.D - d);
            if (a.out_low) store4_low<T>(reinterpret_cast<T *>(a.out_low) + (orow - reinterpret_cast<T *>(a.out)) + d, x, a.D - d);
        }
    if (a.lse && half == 0) a.lse[(long)u.h * a.T * a.group + (long)u.q0 * a.group + row] = l == 0.f ? INFINITY : mc + log2f(l);
}

template <typename T, int DP, int NP, bool WHOLE> __global__ void __launch_bounds__(256, (FwdShape<T, DP, WHOLE>::WAVES)) packed_fwd_kernel(PackedArgs a)
{
    const PackedUnit u = unit_of<false>(a, blockIdx.x);
    if (u.tile * kRows >= u.rows) return;
    constexpr int TERMS = kWeightTerms<T, WHOLE>;
    with_terms<TERMS>(a, u, TERMS == 1 && few_keys(a, u), [](const PackedArgs &b, const PackedUnit &w, auto terms) INLINE { fwd_rows<T, DP, NP, WHOLE, decltype(terms)::value>(b, w); });
}

// The partial results of the workgroups that shared a walk: a workgroup to 16 rows of a tile, a thread to four columns and those 64 further on, four splits
// requested at a time.  Bound: latency (3.1 to 5.4 us).
template <typename T> __global__ void __launch_bounds__(256) packed_join_kernel(PackedArgs a)
{
    const PackedUnit u = unit_of<false>(a, blockIdx.x / 8);
    const int tile_row = blockIdx.x % 8 * 16 + threadIdx.x / 16, row = u.tile * kRows + tile_row;
    const int splits = row_walk(a, u).splits;
    if (row >= u.rows || splits == 1) return;
    const long step = (long)a.tiles * a.Hkv * kRows, first = ((long)u.at * a.Hkv + u.h) * kRows + tile_row;
    const int width = part_width(a.D);
    T *orow = const_cast<T *>(row_at<T>(a.out, a.gs, a, u, row));
    for (int d = threadIdx.x % 16 * 4; d < a.D; d += 64) {
        float all = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < splits; s0 += 4) {
            float2 ml[4];
            float4 y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const long at = first + min(s0 + i, splits - 1) * step;
                ml[i] = *reinterpret_cast<const float2 *>(a.part_ml + at * 2);
                y[i] = *reinterpret_cast<const float4 *>(a.part + at * width + d);
            }
            float top = all;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (s0 + i >= splits) ml[i] = make_float2(-INFINITY, 0.f);
                top = fmaxf(top, ml[i].x);
            }
            const float base = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f(all - base);
            all = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] *= f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (s0 + i >= splits) continue;
                const float g = __builtin_amdgcn_exp2f(ml[i].x - base);
                l = fmaf(ml[i].y, g, l);
                x[0] = fmaf(y[i].x, g, x[0]); x[1] = fmaf(y[i].y, g, x[1]); x[2] = fmaf(y[i].z, g, x[2]); x[3] = fmaf(y[i].w, g, x[3]);
            }
        }
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] *= inv;
        store4<T>(orow + d, x, a.D - d);
        if (a.out_low) store4_low<T>(reinterpret_cast<T *>(a.out_low) + (orow - reinterpret_cast<T *>(a.out)) + d, x, a.D - d);
        if (a.lse && d == 0) a.lse[(long)u.h * a.T * a.group + (long)u.q0 * a.group + row] = l == 0.f ? INFINITY : all + log2f(l);
    }
}

struct FwdPlan { int tiles; Split split; size_t part_bytes, bytes; };
template <typename T> FwdPlan fwd_plan(const d2c_packed_attention_desc &q)
{
    FwdPlan p{};
    p.tiles = tiles_of(q.queries * (q.Hq / q.Hkv), q.sequences);
    const long cus = std::max(d2c_num_cus(), 1);
    pick_width(q.D, fast_kernels(q, false), [&](auto width, auto whole) {
        constexpr int DP = decltype(width)::DP, NP = decltype(width)::NP;
        constexpr bool WHOLE = decltype(whole)::value;
        using Shape = FwdShape<T, DP, WHOLE>;
        p.split = split_walks(q, (long)p.tiles * q.Hkv, cus * resident(reinterpret_cast<const void *>(&packed_fwd_kernel<T, DP, NP, WHOLE>), Shape::LDS), q.keys, Shape::KT,
                              kRows * (part_width(q.D) * 4.0 + 8));
        return 0;
    });
    if (p.split.splits > 1) {
        const size_t lines = (size_t)p.split.splits * p.tiles * q.Hkv * kRows;
        p.part_bytes = d2c_align_up(lines * part_width(q.D) * 4);
        p.bytes = p.part_bytes + d2c_align_up(lines * 8);
    }
    return p;
}
template <typename T> int forward(PackedArgs a, const d2c_packed_attention_desc &q, void *ws, size_t ws_bytes, hipStream_t st)
{
    const FwdPlan p = fwd_plan<T>(q);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 255u))) {
        d2c_set_error("workspace of %zu bytes (256-byte aligned) required, got %zu at %p", p.bytes, ws_bytes, ws);
        return D2C_ERR_WORKSPACE;
    }
    a.tiles = p.tiles; a.splits = p.split.splits; a.chunk = p.split.chunk; a.step = sizeof(T) == 2 ? 64 : 32;
    a.part = (float *)ws; a.part_ml = (float *)((char *)ws + p.part_bytes);
    const int rc = pick_width(q.D, fast_kernels(q, false), [&](auto width, auto whole) {
        constexpr int DP = decltype(width)::DP, NP = decltype(width)::NP;
        constexpr bool WHOLE = decltype(whole)::value;
        constexpr int lds = FwdShape<T, DP, WHOLE>::LDS;
        if (int e = d2c_allow_lds(reinterpret_cast<const void *>(&packed_fwd_kernel<T, DP, NP, WHOLE>), lds, "packed_fwd_kernel")) return e;
        hipLaunchKernelGGL((packed_fwd_kernel<T, DP, NP, WHOLE>), dim3((unsigned)(p.tiles * q.Hkv * p.split.splits)), dim3(256), lds, st, a);
        return d2c_check_launch("packed_fwd_kernel");
    });
    if (rc || p.split.splits == 1) return rc;
    hipLaunchKernelGGL(packed_join_kernel<T>, dim3((unsigned)(p.tiles * q.Hkv * 8)), dim3(256), 0, st, a);
    return d2c_check_launch("packed_join_kernel");
}

}  // namespace

int d2c_packed_attention_check(const d2c_packed_attention_desc *q)
{
    if (!q) { d2c_set_error("packed_attention: null description"); return D2C_ERR_SHAPE; }
    if (q->dtype != D2C_F32 && q->dtype != D2C_BF16) { d2c_set_error("packed_attention: float32 or bfloat16 only"); return D2C_ERR_DTYPE; }
    if (q->sequences < 0 || q->queries < 0 || q->keys < 0 || q->Hq <= 0 || q->Hkv <= 0 || q->D <= 0) {
        d2c_set_error("packed_attention: sizes must not be negative, heads and their size positive");
        return D2C_ERR_SHAPE;
    }
    if (q->Hq % q->Hkv != 0) { d2c_set_error("packed_attention: %d query heads are no multiple of %d key heads", q->Hq, q->Hkv); return D2C_ERR_SHAPE; }
    if (q->D > 128) { d2c_set_error("packed_attention: heads of up to 128 channels, got %d", q->D); return D2C_ERR_UNSUPPORTED; }
    if (q->frame <= 0 || q->frame > (1 << 30)) { d2c_set_error("packed_attention: a frame has 1 to 2^30 tokens, got %d", q->frame); return D2C_ERR_SHAPE; }
    if (!(q->scale > 0.f) || !(q->scale < INFINITY)) { d2c_set_error("packed_attention: scale must be positive and finite"); return D2C_ERR_SHAPE; }
    // (rows, keys and a launch's threads are counted in 32 bits)
    const long most = 1L << 30, group = q->Hq / q->Hkv;
    if (q->queries >= most || q->queries * group >= most || q->keys >= most || q->sequences >= (1 << 20) || q->Hkv >= (1 << 20) ||
        (long)std::max(d2c_packed::tiles_of(q->queries * group, q->sequences), d2c_packed::tiles_of(q->keys, q->sequences)) * q->Hkv >= (1L << 23)) {
        d2c_set_error("packed_attention: too many sequences, tokens or heads");
        return D2C_ERR_SHAPE;
    }
    return D2C_OK;
}

PackedArgs d2c_packed::make_args(const d2c_packed_attention_desc &q, const int32_t *starts, const int32_t *key_starts)
{
    PackedArgs a{};
    for (int i = 0; i < 2; i++) { a.qs[i] = q.q_stride[i]; a.ks[i] = q.k_stride[i]; a.vs[i] = q.v_stride[i]; }
    a.gs[0] = (long)q.Hq * q.D; a.gs[1] = q.D;
    a.T = (int)q.queries; a.Tk = (int)q.keys; a.S = q.sequences; a.Hq = q.Hq; a.Hkv = q.Hkv; a.group = q.Hq / q.Hkv; a.D = q.D; a.causal = q.causal != 0;
    a.by_group = make_fastdiv(a.group); a.frame = make_fastdiv(q.frame);
    a.scale = q.scale; a.scale2 = q.scale * 1.44269504088896340736f;
    a.starts = starts; a.key_starts = key_starts ? key_starts : starts;
    return a;
}

extern "C" size_t d2c_packed_attention_forward_workspace_bytes(const d2c_packed_attention_desc *q)
{
    if (d2c_packed_attention_check(q) != D2C_OK || q->queries == 0) return 0;
    return q->dtype == D2C_BF16 ? fwd_plan<bf16_t>(*q).bytes : fwd_plan<float>(*q).bytes;
}

extern "C" int d2c_packed_attention_forward(const d2c_packed_attention_desc *q, const void *query, const void *key, const void *value,
                                            const int32_t *starts, const int32_t *key_starts, void *out, void *out_low, float *lse,
                                            void *ws, size_t ws_bytes, void *stream)
{
    if (int rc = d2c_packed_attention_check(q)) return rc;
    if (q->queries == 0) return D2C_OK;
    if (!query || !out || (q->keys > 0 && (!key || !value)) || !starts) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    PackedArgs a = make_args(*q, starts, key_starts);
    a.q = query; a.k = key; a.v = value; a.out = out; a.lse = lse;
    a.out_low = q->dtype == D2C_BF16 ? out_low : nullptr;
    return q->dtype == D2C_BF16 ? forward<bf16_t>(a, *q, ws, ws_bytes, (hipStream_t)stream) : forward<float>(a, *q, ws, ws_bytes, (hipStream_t)stream);
}
