// Attention of one map's positions to those of another: backward pass.  Formulas and operand orders: d2c_attention.hpp.
//
// Two kernels, so that every gradient is a sum in one order and none is added up in memory: attn_bwd_q_kernel (a workgroup keeps 128 rows
// and walks over the keys; it also leaves delta of its rows), then attn_bwd_kv_kernel (a workgroup keeps 128 keys, 32 to a wavefront, and walks over the
// rows).  Scores and dp are made in both: 7 products where one kernel would need 5 and would add up dq in memory, in whatever order its workgroups come.  Few rows, or few keys: several workgroups share the
// walk, and attn_bwd_join_kernel adds up their sums.
#include <type_traits>
#include "d2c_attention.hpp"

using namespace d2c_attn;

namespace {

template <typename T, int DP, bool WHOLE> struct QShape {
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;
    using KV = Tile<T, DP, KT, 256, WHOLE>;
    static constexpr int WAVES = sizeof(T) == 2 || DP <= 64 ? 2 : 1;      // to a SIMD
    static constexpr int BUFFERS = 4 * KV::BYTES <= 52 << 10 ? 2 : 1;
    static constexpr int LDS = 2 * BUFFERS * KV::BYTES;
};

// s and dp of a tile of keys, then dq += ds k.  As attn_fwd_kernel: rows along the lanes, ds into the last product's operand in registers, K and V through LDS
// (K read twice, by rows and by columns).  Bound: as there, matrix instructions first (3 products to one exponential).
// Measured, bfloat16: 12960 rows, 25920 keys, 8 heads of 64, 1.04 ms (0.99 PFLOP/s); 1620 rows, 12960 keys (3/4 of them read), 2 samples, 0.13 ms.
// float32: 1417 rows, 3001 keys, 6 heads of 40, 60 us.
template <typename T, int DP, int NP, bool WHOLE> __global__ void __launch_bounds__(256, (QShape<T, DP, WHOLE>::WAVES)) attn_bwd_q_kernel(Args a)
{
    using KV = typename QShape<T, DP, WHOLE>::KV;
    constexpr int P = kTerms<T>, PW = kWeightTerms<T, WHOLE>, ND = DP / 32, NK = kSteps<NP>, KT = QShape<T, DP, WHOLE>::KT;
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int BUFFERS = QShape<T, DP, WHOLE>::BUFFERS;
    constexpr bool END = WHOLE && NP % 2 == 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const Unit unit = unit_of(a);
    const Head hd = unit.head;
    const int tile_row = wave * 32 + (lane & 31), row = unit.tile * 128 + tile_row;
    const bool live = row < a.rows;
    const int keys = keys_of(a, hd.n), tiles = (keys + KT - 1) / KT;
    const bool alone = one_key(a, hd.n, keys);
    const int t1 = alone ? 0 : (int)((long)tiles * (unit.split + 1) / unit.splits);
    int t = (int)((long)tiles * unit.split / unit.splits);

    KV k, v;
    const KeyTiles<T, KV, KT, 1, WHOLE> source(a, hd);
    bool b = false;
    auto ask = [&](int k0) INLINE { const int key = k0 + lane; b = lane < KT && key < keys && (!a.mask || a.mask[(long)hd.n * a.Lk + key]); };
    uint64_t next[1] = {0};
    auto request = [&](int tile) INLINE { source.request(a, k, v, tile, next); };
    if (t < t1) {
        ask(t * KT);
        next[0] = __ballot(b);
        request(t);
        ask((t + 1) * KT);
    }
    Frag<P> q[NK], g[NK];
    float delta = 0.f;
    {
        const int r = min(row, a.rows - 1);
        const T *qr = row_at<T>(a.q, a.qs, a, hd, r), *gr = row_at<T>(a.g, a.gs, a, hd, r), *orow = row_at<T>(a.o, a.gs, a, hd, r);
#pragma unroll
        for (int i = 0; i < NK; i++) {
            const int d = i * 16 + half * 8;
            q[i] = terms_of<T>(load8_of<WHOLE, T>(qr, d, a.D, live));
            const Raw8<T> x = load8_of<WHOLE, T>(gr, d, a.D, live), y = load8_of<WHOLE, T>(orow, d, a.D, live);
            g[i] = terms_of<T>(x);
            float xf[8], yf[8];
            floats_of<T>(x, xf);
            floats_of<T>(y, yf);
            if (a.o_low) {
                float lf[8];
                floats_of<T>(load8_of<WHOLE, T>(row_at<T>(a.o_low, a.gs, a, hd, r), d, a.D, live), lf);
#pragma unroll
                for (int j = 0; j < 8; j++) yf[j] += lf[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) delta = fmaf(xf[j], yf[j], delta);
        }
    }
    delta = half_sum(delta);
    const float lse = live ? a.lse[hd.nh * a.rows + row] : INFINITY;
    if (live && unit.split == 0 && half == 0) a.delta[hd.nh * a.rows + row] = delta;
    // (a row with one key has gradients of 0, but none where its weight, its output or the output's gradient is no finite number)
    const float none = alone && !(lse == lse && fabsf(delta) < INFINITY) ? NAN : 0.f;
    f32x16 dq[ND];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) dq[i][r] = none;
    const float c = a.scale2;
    int buffer = 0;

    for (; t < t1; t++) {
        const uint64_t now = next[0];
        unsigned char *s_k = lds + (BUFFERS == 2 ? buffer * 2 * KV::BYTES : 0), *s_v = s_k + KV::BYTES;
        buffer ^= 1;
        if constexpr (BUFFERS == 1) __syncthreads();
        k.template store<END>(s_k, a.D);
        v.template store<false>(s_v, a.D);      // (an infinite value leaves no gradient of its row defined, whatever it meets)
        __syncthreads();
        if (t + 1 < t1) {
            next[0] = __ballot(b);
            request(t + 1);
            ask((t + 2) * KT);
        }
        if (now == 0) continue;
#pragma unroll
        for (int i = 0; i < KT / 32; i++) {
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = dp[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NK; ks++) {
                mma(s, KV::rows(s_k, i * 32 + (lane & 31), ks, half), q[ks]);
                mma(dp, KV::rows(s_v, i * 32 + (lane & 31), ks, half), g[ks]);
            }
            const uint32_t there = (uint32_t)(now >> (i * 32));
            if (there != 0xffffffffu) {
                const uint32_t w = there >> (half * 4);
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!((w >> (8 * (r / 4) + r % 4)) & 1)) s[r] = -INFINITY;
            }
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; r++) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (dp[r] - delta);
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                const Frag<PW> f = make_frag<PW, MADE>(ds + kk * 8);
#pragma unroll
                for (int d = 0; d < ND; d++) mma(dq[d], KV::columns(s_k, i * 32 + kk * 16, d * 32, lane), f);
            }
        }
    }
    if (!live) return;
    if (unit.splits > 1) {
        float *p = a.part + (((long)unit.split * a.shared + unit.part) * 128 + tile_row) * part_width(a.D);
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int d = i * 32 + j * 8 + half * 4;
                const float x[4] = {dq[i][j * 4], dq[i][j * 4 + 1], dq[i][j * 4 + 2], dq[i][j * 4 + 3]};
                store4<float>(p + d, x, a.D - d);
            }
        return;
    }
    T *out = const_cast<T *>(row_at<T>(a.gq, a.gs, a, hd, row));
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + j * 8 + half * 4;
            const float x[4] = {dq[i][j * 4] * a.scale, dq[i][j * 4 + 1] * a.scale, dq[i][j * 4 + 2] * a.scale, dq[i][j * 4 + 3] * a.scale};
            store4<T>(out + d, x, a.D - d);
        }
}

template <typename T, int DP, bool WHOLE> struct KvShape {
    // V of the workgroup's keys in LDS where registers do not hold it beside the sums
    static constexpr bool V_LDS = sizeof(T) == 2 && DP == 128;
    static constexpr int WAVES = sizeof(T) == 2 || DP <= 64 ? 2 : 1;      // to a SIMD
    using V = Tile<T, DP, 128, 256, false>;      // (zeros behind a row's end: the other operand has its last piece again there)
    static constexpr int V_BYTES = V_LDS ? V::BYTES : 0;
    static constexpr int RT = sizeof(T) == 2 && DP <= 64 ? 64 : 32;
    using QG = Tile<T, DP, RT, 256, WHOLE>;
    static constexpr int BYTES = 2 * QG::BYTES + 2 * RT * 4, BUFFERS = 2 * BYTES <= 52 << 10 && !V_LDS ? 2 : 1;
    static constexpr int LDS = BUFFERS * BYTES + V_BYTES;
};

// Keys along the lanes, their K and V in registers from first to last; queries and grad_out of a tile of rows through LDS, each read by rows (s, dp) and by
// columns (dk, dv).  dp starts from -delta, one subtraction less to a score.  K and V in LDS, too, would make room for a third workgroup to a compute unit, and takes
// 1.5 times as long at 64 channels: the LDS is read six times a tile then.  A mask costs nothing and saves nothing here: rows of tiles whose keys are all not to be read are walked
// over, too (behind a sample's length they are not).  Bound: matrix instructions (4 products to one exponential), behind them LDS.
// Measured, bfloat16: 12960 rows, 25920 keys, 8 heads of 64, 1.38 ms (1.0 PFLOP/s); 1620 rows, 12960 keys (3/4 of them read), 2 samples, 0.21 ms.
// float32: 1417 rows, 3001 keys, 6 heads of 40, 72 us.
template <typename T, int DP, int NP, bool WHOLE> __global__ void __launch_bounds__(256, (KvShape<T, DP, WHOLE>::WAVES)) attn_bwd_kv_kernel(Args a)
{
    using QG = typename KvShape<T, DP, WHOLE>::QG;
    constexpr int P = kTerms<T>, PW = kWeightTerms<T, WHOLE>, ND = DP / 32, NK = kSteps<NP>, RT = KvShape<T, DP, WHOLE>::RT;
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int BUFFERS = KvShape<T, DP, WHOLE>::BUFFERS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const Unit unit = unit_of(a);
    const Head hd = unit.head;
    const int tile_key = wave * 32 + (lane & 31), keys = keys_of(a, hd.n), key0 = unit.tile * 128, key = key0 + tile_key;
    const bool live = key < keys && (!a.mask || a.mask[(long)hd.n * a.Lk + key]), alone = one_key(a, hd.n, keys);
    const int tiles = (a.rows + RT - 1) / RT;
    const int t1 = key0 < keys ? (int)((long)tiles * (unit.split + 1) / unit.splits) : 0;
    int t = (int)((long)tiles * unit.split / unit.splits);

    QG q, g;
    const T *qb = row_at<T>(a.q, a.qs, a, hd, 0), *gb = row_at<T>(a.g, a.gs, a, hd, 0);
    // (tiles that begin with a position's first head: the places of their rows are the same from tile to tile)
    const bool uniform = RT % a.group == 0;
    unsigned qoff[WHOLE ? QG::PER : 1], goff[WHOLE ? QG::PER : 1];
    auto places = [&](unsigned (&qo)[WHOLE ? QG::PER : 1], unsigned (&go)[WHOLE ? QG::PER : 1], int r0) INLINE {
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < QG::PER; i++) {
                const unsigned row = min(r0 + QG::row_of(i), a.rows - 1), pos = row / (unsigned)a.group, head = row - pos * a.group, d = QG::column_of(i, a.D);
                qo[i] = (pos * (unsigned)a.qs[1] + head * (unsigned)a.qs[2] + d) * (unsigned)sizeof(T);
                go[i] = (pos * (unsigned)a.gs[1] + head * (unsigned)a.gs[2] + d) * (unsigned)sizeof(T);
            }
        }
    };
    places(qoff, goff, 0);
    float stat = 0.f;
    auto request = [&](int tile) INLINE {
        const int r0 = tile * RT;
        // (rows behind the last one repeat it: their weights are 0, by a sum of +infinity, and their gradients are made 0 on the way to LDS)
        if constexpr (WHOLE) {
            if (uniform && r0 + RT <= a.rows) {
                q.load_at(qb + (long)(r0 / a.group) * a.qs[1], qoff);
                g.load_at(gb + (long)(r0 / a.group) * a.gs[1], goff);
            } else {
                unsigned qo[QG::PER], go[QG::PER];
                places(qo, go, r0);
                q.load_at(qb, qo);
                g.load_at(gb, go);
            }
        } else {
            q.load(a.D, [&](int i) INLINE { return row_at<T>(a.q, a.qs, a, hd, min(r0 + i, a.rows - 1)); });
            g.load(a.D, [&](int i) INLINE { return row_at<T>(a.g, a.gs, a, hd, min(r0 + i, a.rows - 1)); });
        }
        if (threadIdx.x < 2 * RT) {
            const bool first = threadIdx.x < RT;
            const int r = r0 + (first ? threadIdx.x : threadIdx.x - RT);
            stat = r < a.rows ? (first ? a.lse[hd.nh * a.rows + r] : -a.delta[hd.nh * a.rows + r]) : (first ? INFINITY : 0.f);
        }
    };
    if (t < t1) request(t);
    using Shape = KvShape<T, DP, WHOLE>;
    Frag<P> k[NK], v[Shape::V_LDS ? 1 : NK];
    unsigned char *s_v = lds + BUFFERS * Shape::BYTES;
    if constexpr (Shape::V_LDS) {
        typename Shape::V tile;
        const T *vb = reinterpret_cast<const T *>(a.v) + hd.n * a.vs[0] + hd.h * a.vs[2];
        tile.load(a.D, [&](int i) INLINE { return vb + (long)min(key0 + i, a.Lk - 1) * a.vs[1]; });
        tile.template store<false>(s_v, a.D);      // (a key that is not to be read: a column of its own, see below)
    }
    {
        const long at = min(key, a.Lk - 1);
        const T *kr = reinterpret_cast<const T *>(a.k) + hd.n * a.ks[0] + hd.h * a.ks[2] + at * a.ks[1];
        const T *vr = reinterpret_cast<const T *>(a.v) + hd.n * a.vs[0] + hd.h * a.vs[2] + at * a.vs[1];
#pragma unroll
        for (int i = 0; i < NK; i++) {
            const int d = i * 16 + half * 8;
            k[i] = terms_of<T>(load8_of<WHOLE, T>(kr, d, a.D, live));
            if constexpr (!Shape::V_LDS) v[i] = terms_of<T>(load8_of<WHOLE, T>(vr, d, a.D, live));
        }
    }
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) dk[i][r] = dv[i][r] = 0.f;
    const float c = a.scale2;
    int buffer = 0;

    for (; t < t1; t++) {
        unsigned char *s_q = lds + (BUFFERS == 2 ? buffer * KvShape<T, DP, WHOLE>::BYTES : 0), *s_g = s_q + QG::BYTES;
        float *s_lse = reinterpret_cast<float *>(s_q + 2 * QG::BYTES), *s_delta = s_lse + RT;
        buffer ^= 1;
        if constexpr (BUFFERS == 1) __syncthreads();
        if (t * RT + RT > a.rows) g.zero_rows([&](int i) INLINE { return t * RT + i >= a.rows; });
        q.template store<false>(s_q, a.D);      // (an infinite query has no defined weights, an infinite gradient no defined ds)
        g.template store<false>(s_g, a.D);
        if (threadIdx.x < 2 * RT) s_lse[threadIdx.x] = stat;
        __syncthreads();
        if (t + 1 < t1) request(t + 1);
#pragma unroll
        for (int i = 0; i < RT / 32; i++) {
            f32x16 s, dp;      // (dp starts from -delta of its rows)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 de = *reinterpret_cast<const float4 *>(s_delta + i * 32 + j * 8 + half * 4);
                dp[j * 4] = de.x; dp[j * 4 + 1] = de.y; dp[j * 4 + 2] = de.z; dp[j * 4 + 3] = de.w;
            }
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NK; ks++) {
                mma(s, QG::rows(s_q, i * 32 + (lane & 31), ks, half), k[ks]);
                if constexpr (Shape::V_LDS) mma(dp, QG::rows(s_g, i * 32 + (lane & 31), ks, half), Shape::V::rows(s_v, tile_key, ks, half));
                else mma(dp, QG::rows(s_g, i * 32 + (lane & 31), ks, half), v[ks]);
            }
            float p[16], ds[16];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 ls = *reinterpret_cast<const float4 *>(s_lse + i * 32 + j * 8 + half * 4);
                const float lr[4] = {ls.x, ls.y, ls.z, ls.w};
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    p[j * 4 + r] = __builtin_amdgcn_exp2f(fmaf(s[j * 4 + r], c, -lr[r]));
                    ds[j * 4 + r] = p[j * 4 + r] * dp[j * 4 + r];
                }
            }
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                const Frag<PW> pf = make_frag<PW, WEIGHTS>(p + kk * 8), df = make_frag<PW, MADE>(ds + kk * 8);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    mma(dv[d], QG::columns(s_g, i * 32 + kk * 16, d * 32, lane), pf);
                    mma(dk[d], QG::columns(s_q, i * 32 + kk * 16, d * 32, lane), df);
                }
            }
        }
    }
    if (key >= a.Lk) return;
    // (a key that is not to be read: a column of the accumulators of its own, whatever is in it)
    const float fk = unit.splits > 1 ? 1.f : a.scale;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + j * 8 + half * 4;
            float x[4], y[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r] = live ? dk[i][j * 4 + r] * fk : 0.f;
                if (alone && x[r] == x[r]) x[r] = 0.f;
                y[r] = live ? dv[i][j * 4 + r] : 0.f;
            }
            if (unit.splits > 1) {
                store4<float>(a.part + (((2L * unit.split) * a.shared + unit.part) * 128 + tile_key) * part_width(a.D) + d, x, a.D - d);
                store4<float>(a.part + (((2L * unit.split + 1) * a.shared + unit.part) * 128 + tile_key) * part_width(a.D) + d, y, a.D - d);
            } else {
                const long at = (((long)hd.n * a.Lk + key) * a.Hkv + hd.h) * a.D + d;
                if (a.gk) store4<T>(reinterpret_cast<T *>(a.gk) + at, x, a.D - d);
                if (a.gv) store4<T>(reinterpret_cast<T *>(a.gv) + at, y, a.D - d);
            }
        }
}

// Sums of the workgroups that shared a walk: part [splits][1 or 2][shared][128][D].  A thread takes four of a row's columns, four splits requested at a time.
// Bound: memory.  26624 rows of 64 columns 9.2 us, 13.3 as a thread to a column.
template <typename T, bool KV> __global__ void __launch_bounds__(256) attn_bwd_join_kernel(Args a)
{
    const int total = a.shared * 128, pieces = part_width(a.D) / 4;
    const long index = (long)blockIdx.x * 256 + threadIdx.x;
    const int line = (int)(index / pieces), d = (int)(index - (long)line * pieces) * 4;
    if (line >= total) return;
    const int which = KV ? blockIdx.y : 0;
    if (KV && !(which ? a.gv : a.gk)) return;
    const int unit = a.whole + line / 128, heads = a.N * a.Hkv, tile = unit / heads, nh = unit - tile * heads;
    const int i = tile * 128 + line % 128, n = nh / a.Hkv;
    if (i >= (KV ? a.Lk : a.rows)) return;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.splits; s0 += 4) {
        float4 y[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            y[u] = *reinterpret_cast<const float4 *>(a.part + (((long)min(s0 + u, a.splits - 1) * (KV ? 2 : 1) + which) * total + line) * part_width(a.D) + d);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (s0 + u >= a.splits) continue;
            x[0] += y[u].x; x[1] += y[u].y; x[2] += y[u].z; x[3] += y[u].w;
        }
    }
    if (which == 0) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] *= a.scale;
    }
    const Head hd{n, nh - n * a.Hkv, nh};
    if constexpr (KV)
        store4<T>(reinterpret_cast<T *>(which ? a.gv : a.gk) + (((long)n * a.Lk + i) * a.Hkv + hd.h) * a.D + d, x, a.D - d);
    else
        store4<T>(const_cast<T *>(row_at<T>(a.gq, a.gs, a, hd, i)) + d, x, a.D - d);
}

// delta alone, where the queries' gradient is not wanted: one wavefront to a row (and to the rows a launch's wavefronts further on, so that its threads can be
// counted in 32 bits)
constexpr long kDeltaBlocks = 1L << 20;
template <typename T> __global__ void __launch_bounds__(256) attn_delta_kernel(Args a)
{
    const long total = (long)a.N * a.Hkv * a.rows;
    const int lane = threadIdx.x & 63;
    for (long at = (long)blockIdx.x * 4 + (threadIdx.x >> 6); at < total; at += 4L * gridDim.x) {
        const long nh = at / a.rows;
        const int n = (int)(nh / a.Hkv);
        const Head hd{n, (int)(nh - (long)n * a.Hkv), nh};
        const T *g = row_at<T>(a.g, a.gs, a, hd, (int)(at - nh * a.rows)), *o = row_at<T>(a.o, a.gs, a, hd, (int)(at - nh * a.rows));
        const T *low = a.o_low ? row_at<T>(a.o_low, a.gs, a, hd, (int)(at - nh * a.rows)) : nullptr;
        float x = 0.f;
        for (int d = lane; d < a.D; d += 64) x = fmaf(elem_to_f32<T>(g[d]), elem_to_f32<T>(o[d]) + (low ? elem_to_f32<T>(low[d]) : 0.f), x);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
        if (lane == 0) a.delta[at] = x;
    }
}

struct BwdPlan { Walks q, kv; size_t delta_bytes, bytes; };
template <typename T> BwdPlan bwd_plan(const d2c_attention_desc &q)
{
    BwdPlan p;
    const long rows = (long)q.Lq * (q.Hq / q.Hkv), heads = (long)q.N * q.Hkv, cus = std::max(d2c_num_cus(), 1);
    const double part = 128.0 * part_width(q.D) * 4, limit = part_limit(q), slow = sizeof(T) == 2 ? 1 : 3;
    for_width<T, true>(q, [&](auto width, auto whole) {
        constexpr int DP = decltype(width)::DP, NP = decltype(width)::NP;
        constexpr bool WHOLE = decltype(whole)::value;
        using Q = QShape<T, DP, WHOLE>;
        using KV = KvShape<T, DP, WHOLE>;
        // (a step with every place taken, 64 channels: 64 keys 2.4 us, 64 rows 2.8)
        p.q = plan_walks(heads * ((rows + 127) / 128), (q.Lk + Q::KT - 1) / Q::KT,
                         cus * resident(reinterpret_cast<const void *>(&attn_bwd_q_kernel<T, DP, NP, WHOLE>), Q::LDS), 2.4 * Q::KT / 64 * DP / 64 * slow, part, limit);
        p.kv = plan_walks(heads * ((q.Lk + 127) / 128), (rows + KV::RT - 1) / KV::RT,
                          cus * resident(reinterpret_cast<const void *>(&attn_bwd_kv_kernel<T, DP, NP, WHOLE>), KV::LDS), 2.8 * KV::RT / 64 * DP / 64 * slow, 2 * part, limit);
        return 0;
    });
    p.delta_bytes = d2c_align_up((size_t)heads * rows * 4);
    const size_t unit = (size_t)128 * part_width(q.D) * 4;
    p.bytes = p.delta_bytes + d2c_align_up(std::max(p.q.shared * p.q.splits * unit, 2 * p.kv.shared * p.kv.splits * unit));
    return p;
}

template <typename T, int DP, int NP, bool WHOLE> int launch_bwd(Args a, const BwdPlan &p, hipStream_t st)
{
    if (a.Lq > 0 && !a.gq && (a.gk || a.gv)) {
        hipLaunchKernelGGL(attn_delta_kernel<T>, dim3((unsigned)std::min(((long)a.N * a.Hkv * a.rows + 3) / 4, kDeltaBlocks)), dim3(256), 0, st, a);
        if (int rc = d2c_check_launch("attn_delta_kernel")) return rc;
    } else if (a.Lq > 0 && a.gq) {
        constexpr int lds = QShape<T, DP, WHOLE>::LDS;
        if (int rc = d2c_allow_lds(reinterpret_cast<const void *>(&attn_bwd_q_kernel<T, DP, NP, WHOLE>), lds, "attn_bwd_q_kernel")) return rc;
        set_walks(a, p.q);
        hipLaunchKernelGGL((attn_bwd_q_kernel<T, DP, NP, WHOLE>), dim3(workgroups(p.q)), dim3(256), lds, st, a);
        if (int rc = d2c_check_launch("attn_bwd_q_kernel")) return rc;
        if (p.q.shared > 0) {
            hipLaunchKernelGGL((attn_bwd_join_kernel<T, false>), dim3((unsigned)(((long)p.q.shared * 128 * (part_width(a.D) / 4) + 255) / 256)), dim3(256), 0, st, a);
            if (int rc = d2c_check_launch("attn_bwd_join_kernel")) return rc;
        }
    }
    if (a.Lk == 0 || !(a.gk || a.gv)) return D2C_OK;
    constexpr int lds = KvShape<T, DP, WHOLE>::LDS;
    if (int rc = d2c_allow_lds(reinterpret_cast<const void *>(&attn_bwd_kv_kernel<T, DP, NP, WHOLE>), lds, "attn_bwd_kv_kernel")) return rc;
    set_walks(a, p.kv);
    hipLaunchKernelGGL((attn_bwd_kv_kernel<T, DP, NP, WHOLE>), dim3(workgroups(p.kv)), dim3(256), lds, st, a);
    if (int rc = d2c_check_launch("attn_bwd_kv_kernel")) return rc;
    if (p.kv.shared == 0) return D2C_OK;
    hipLaunchKernelGGL((attn_bwd_join_kernel<T, true>), dim3((unsigned)(((long)p.kv.shared * 128 * (part_width(a.D) / 4) + 255) / 256), 2), dim3(256), 0, st, a);
    return d2c_check_launch("attn_bwd_join_kernel");
}
template <typename T> int backward(Args a, const d2c_attention_desc &q, void *ws, size_t ws_bytes, hipStream_t st)
{
    const BwdPlan p = bwd_plan<T>(q);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 255u))) {
        d2c_set_error("workspace of %zu bytes (256-byte aligned) required, got %zu at %p", p.bytes, ws_bytes, ws);
        return D2C_ERR_WORKSPACE;
    }
    a.delta = (float *)ws; a.part = (float *)((char *)ws + p.delta_bytes);
    return for_width<T, true>(q, [&](auto width, auto whole) { return launch_bwd<T, decltype(width)::DP, decltype(width)::NP, decltype(whole)::value>(a, p, st); });
}

}  // namespace

extern "C" size_t d2c_attention_backward_workspace_bytes(const d2c_attention_desc *q)
{
    if (d2c_attention_check(q) != D2C_OK || q->N == 0) return 0;
    return q->dtype == D2C_BF16 ? bwd_plan<bf16_t>(*q).bytes : bwd_plan<float>(*q).bytes;
}

extern "C" int d2c_attention_backward(const d2c_attention_desc *q, const void *grad_out, const void *query, const void *key,
                                      const void *value, const int32_t *key_lengths, const uint8_t *key_mask, const void *out,
                                      const void *out_low, const float *lse, void *grad_query, void *grad_key, void *grad_value, void *ws,
                                      size_t ws_bytes, void *stream)
{
    if (int rc = d2c_attention_check(q)) return rc;
    if (q->N == 0 || (q->Lq == 0 && q->Lk == 0)) return D2C_OK;
    if ((q->Lq > 0 && (!grad_out || !query || !out || !lse)) || (q->Lk > 0 && (!key || !value))) {
        d2c_set_error("null tensor pointer");
        return D2C_ERR_SHAPE;
    }
    Args a = make_args(*q);
    a.g = grad_out; a.q = query; a.k = key; a.v = value; a.lengths = key_lengths; a.mask = key_mask; a.o = out;
    a.o_low = q->dtype == D2C_BF16 ? out_low : nullptr;
    a.lse = const_cast<float *>(lse);
    a.gq = grad_query; a.gk = grad_key; a.gv = grad_value;
    return q->dtype == D2C_BF16 ? backward<bf16_t>(a, *q, ws, ws_bytes, (hipStream_t)stream) : backward<float>(a, *q, ws, ws_bytes, (hipStream_t)stream);
}
