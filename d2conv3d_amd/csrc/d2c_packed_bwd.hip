// Attention inside sequences that lie behind each other: backward pass.  Shared parts: d2c_packed.hpp.
//
// Two kernels, so that every gradient is a sum in one order and none is added up in memory: packed_bwd_q_kernel (a workgroup keeps 128 rows and walks over the keys that
// they read; it leaves delta of its rows), then packed_bwd_kv_kernel (a workgroup keeps 128 keys, 32 to a wavefront, and walks over the rows that read any of them).
// A row that reads one key has exact zeros as gradients of its score, which two sums of the same terms in different orders would not leave.
#include "d2c_packed.hpp"

using namespace d2c_packed;

namespace {

template <typename T, int DP, bool WHOLE> struct QShape {
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;
    using KV = Tile<T, DP, KT, 256, WHOLE>;
    static constexpr int WAVES = sizeof(T) == 2 || DP <= 64 ? 2 : 1;      // to a SIMD
    static constexpr int BUFFERS = 4 * KV::BYTES <= 52 << 10 ? 2 : 1;
    static constexpr int LDS = 2 * BUFFERS * KV::BYTES;
};

// s and dp of a tile of keys, then dq += ds k.  As attn_bwd_q_kernel: rows along the lanes, ds into the last product's operand in registers, K and V through LDS (K read
// twice, by rows and by columns; where it holds infinities or NaN and some rows do not read all of the tile, it is cleaned in LDS between the two).  Bound: matrix instructions (3 products to
// one exponential).  Measured, bfloat16: one sequence of 25920, 8 heads of 64 that share 2, 1.07 ms (0.96 PFLOP/s); six of up to 12960 in frames, 8 heads of 64, 0.98 ms (0.89).  float32: three of up to
// 1417, 6 heads of 40, 34 us and the join 4.8.
template <typename T, int DP, int NP, bool WHOLE, int PW> D2C_DEV void bwd_rows(const PackedArgs &a, const PackedUnit &u)
{
    using Shape = QShape<T, DP, WHOLE>;
    using KV = typename Shape::KV;
    constexpr int P = kTerms<T>, ND = DP / 32, NK = kSteps<NP>, KT = Shape::KT, BUFFERS = Shape::BUFFERS;
    constexpr bool END = WHOLE && NP % 2 == 1;
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ int s_bad[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, row0 = u.tile * kRows;
    const int tile_row = wave * 32 + (lane & 31), row = row0 + tile_row;
    const bool live = row < u.rows;
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
    Frag<P> q[NK], g[NK];
    float delta = 0.f;
    {
        const int r = min(row, u.rows - 1);
        const T *qr = row_at<T>(a.q, a.qs, a, u, r), *gr = row_at<T>(a.g, a.gs, a, u, r), *orow = row_at<T>(a.o, a.gs, a, u, r);
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
                floats_of<T>(load8_of<WHOLE, T>(row_at<T>(a.o_low, a.gs, a, u, r), d, a.D, live), lf);
#pragma unroll
                for (int j = 0; j < 8; j++) yf[j] += lf[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) delta = fmaf(xf[j], yf[j], delta);
        }
    }
    delta = half_sum(delta);
    const long stat = (long)u.h * a.T * a.group + (long)u.q0 * a.group + row;
    const float lse = live ? a.lse[stat] : INFINITY;
    if (live && u.split == 0 && half == 0) a.delta[stat] = delta;
    f32x16 dq[ND];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) dq[i][r] = 0.f;
    const float c = a.scale2, alone = lim == 1 ? 0.f : 1.f;
    int buffer = 0;
    bool any_bad = false;

    for (; t < t1; t++) {
        unsigned char *s_k = lds + (BUFFERS == 2 ? buffer * 2 * KV::BYTES : 0), *s_v = s_k + KV::BYTES;
        const bool masked = t * KT + KT > least;
        if constexpr (BUFFERS == 1) __syncthreads();
        if (masked) {
            const int left = u.lk - t * KT;
            k.zero_rows([&](int i) INLINE { return i >= left; });
            const bool bad = __any(not_finite<T>(k));
            if (lane == 0) s_bad[buffer][wave] = bad;
        }
        k.template store<END>(s_k, a.D);
        v.template store<false>(s_v, a.D);
        __syncthreads();
        if (t + 1 < t1) source.request(a, k, v, t + 1, u.lk - (t + 1) * KT);
        const bool bad = masked && (s_bad[buffer][0] | s_bad[buffer][1] | s_bad[buffer][2] | s_bad[buffer][3]);
        any_bad = any_bad || bad;
        buffer ^= 1;
        if (t * KT >= wave_most && !bad) continue;      // (all meet at the barriers below)
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
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; r++) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (dp[r] - delta);
            const int key0 = t * KT + i * 32;
            if (key0 + 32 > wave_least) {      // (so it is where a row reads one key)
                const int left = lim - (key0 + half * 4);
#pragma unroll
                for (int r = 0; r < 16; r++) ds[r] = 8 * (r / 4) + r % 4 < left ? ds[r] * alone : 0.f;
            }
            if (bad) {
                __syncthreads();
                clean_rows<KV>(s_k, i * 32);
                __syncthreads();
            }
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                const Frag<PW> f = make_frag<PW, MADE>(ds + kk * 8);
#pragma unroll
                for (int d = 0; d < ND; d++) mma(dq[d], KV::columns(s_k, i * 32 + kk * 16, d * 32, lane), f);
            }
        }
    }
    if (any_bad)
        take_in<T, true>(dq, a.D, max(least / KT, t0) * KT, min(t1 * KT, wave_most), [&](int j) INLINE { return source.kb + (long)j * source.ks; },
                         [&](int j) INLINE { return j < lim; });
    if (!live) return;
    if (walk.splits > 1) {
        float *p = a.part + ((((long)u.split * a.tiles + u.at) * a.Hkv + u.h) * kRows + tile_row) * part_width(a.D);
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
    T *out = const_cast<T *>(row_at<T>(a.gq, a.gs, a, u, row));
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + j * 8 + half * 4;
            const float x[4] = {dq[i][j * 4] * a.scale, dq[i][j * 4 + 1] * a.scale, dq[i][j * 4 + 2] * a.scale, dq[i][j * 4 + 3] * a.scale};
            store4<T>(out + d, x, a.D - d);
        }
}

template <typename T, int DP, int NP, bool WHOLE> __global__ void __launch_bounds__(256, (QShape<T, DP, WHOLE>::WAVES)) packed_bwd_q_kernel(PackedArgs a)
{
    const PackedUnit u = unit_of<false>(a, blockIdx.x);
    if (u.tile * kRows >= u.rows) return;
    constexpr int TERMS = kWeightTerms<T, WHOLE>;
    with_terms<TERMS>(a, u, TERMS == 1 && few_keys(a, u), [](const PackedArgs &b, const PackedUnit &w, auto terms) INLINE { bwd_rows<T, DP, NP, WHOLE, decltype(terms)::value>(b, w); });
}

template <typename T, int DP, bool WHOLE> struct KvShape {
    // V of the workgroup's keys in LDS where registers do not hold it beside the sums
    static constexpr bool V_LDS = sizeof(T) == 2 && DP == 128;
    static constexpr int WAVES = sizeof(T) == 2 || DP <= 64 ? 2 : 1;      // to a SIMD
    using V = Tile<T, DP, 128, 256, false>;      // (zeros behind a row's end: the other operand has its last piece again there)
    static constexpr int V_BYTES = V_LDS ? V::BYTES : 0;
    static constexpr int RT = sizeof(T) == 2 && DP <= 64 ? 64 : 32;
    using QG = Tile<T, DP, RT, 256, WHOLE>;
    static constexpr int BYTES = 2 * QG::BYTES + 3 * RT * 4, BUFFERS = 2 * BYTES <= 52 << 10 && !V_LDS ? 2 : 1;
    static constexpr int LDS = BUFFERS * BYTES + V_BYTES;
};

// Keys along the lanes, their K and V in registers from first to last; queries and grad_out of a tile of rows through LDS, each read by rows (s, dp) and by columns
// (dk, dv).  dp starts from -delta.  As attn_bwd_kv_kernel; the walk begins with the first row that reads a key of the tile.  Bound: matrix instructions (4 products to one exponential), behind
// them LDS.  Measured, bfloat16: one sequence of 25920, 8 heads of 64 that share 2, 1.49 ms and the join 23 us (0.93 PFLOP/s; 3.1 ms before walks were cut in pieces, the first keys' being as long
// as the whole sequence); six of up to 12960 in frames, 8 heads of 64, 1.21 ms (0.96).  float32: three of up to 1417, 6 heads of 40, 42 us and the join 5.4.
template <typename T, int DP, int NP, bool WHOLE, int PW> D2C_DEV void bwd_keys(const PackedArgs &a, const PackedUnit &u)
{
    using Shape = KvShape<T, DP, WHOLE>;
    using QG = typename Shape::QG;
    constexpr int P = kTerms<T>, ND = DP / 32, NK = kSteps<NP>, RT = Shape::RT, BUFFERS = Shape::BUFFERS;
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ int s_bad[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, key0 = u.tile * kRows;
    const int tile_key = wave * 32 + (lane & 31), key = key0 + tile_key, keys_end = min(key0 + kRows, u.lk);
    const bool live = key < u.lk;
    const Walk walk = key_walk(a, u);
    if (u.split >= walk.splits) return;
    const int t1 = walk.first + (int)((long)walk.steps * (u.split + 1) / walk.splits);
    const int t0 = walk.first + (int)((long)walk.steps * u.split / walk.splits);
    int t = t0;

    QG q, g;
    // (tiles that begin with a position's first head: the places of their rows are the same from tile to tile)
    const bool uniform = RT % a.group == 0;
    const T *qb = reinterpret_cast<const T *>(a.q) + (long)u.q0 * a.qs[0] + (long)u.h * a.group * a.qs[1];
    const T *gb = reinterpret_cast<const T *>(a.g) + (long)u.q0 * a.gs[0] + (long)u.h * a.group * a.gs[1];
    unsigned qoff[WHOLE ? QG::PER : 1], goff[WHOLE ? QG::PER : 1];
    auto places = [&](unsigned (&qo)[WHOLE ? QG::PER : 1], unsigned (&go)[WHOLE ? QG::PER : 1], int r0, int pos0) INLINE {
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < QG::PER; i++) {
                const int row = min(r0 + QG::row_of(i), u.rows - 1), pos = fdiv(row, a.by_group), d = QG::column_of(i, a.D);
                const unsigned at = pos - pos0, head = row - pos * a.group;
                qo[i] = (at * (unsigned)a.qs[0] + head * (unsigned)a.qs[1] + d) * (unsigned)sizeof(T);
                go[i] = (at * (unsigned)a.gs[0] + head * (unsigned)a.gs[1] + d) * (unsigned)sizeof(T);
            }
        }
    };
    const long stats = (long)u.h * a.T * a.group + (long)u.q0 * a.group;
    float stat = 0.f;
    auto request = [&](int tile) INLINE {
        const int r0 = tile * RT;
        // (rows behind the last one repeat it: their weights are 0, by a sum of +infinity, and their gradients are made 0 on the way to LDS)
        if constexpr (WHOLE) {
            const int pos0 = fdiv(r0, a.by_group);
            const T *qt = qb + (long)pos0 * a.qs[0], *gt = gb + (long)pos0 * a.gs[0];
            if (!uniform || r0 + RT > u.rows) {
                unsigned qo[QG::PER], go[QG::PER];
                places(qo, go, r0, pos0);
                q.load_at(qt, qo);
                g.load_at(gt, go);
            } else {
                q.load_at(qt, qoff);
                g.load_at(gt, goff);
            }
        } else {
            q.load(a.D, [&](int i) INLINE { return row_at<T>(a.q, a.qs, a, u, min(r0 + i, u.rows - 1)); });
            g.load(a.D, [&](int i) INLINE { return row_at<T>(a.g, a.gs, a, u, min(r0 + i, u.rows - 1)); });
        }
        if (threadIdx.x < 3 * RT) {
            const int which = threadIdx.x / RT, r = r0 + (int)threadIdx.x - which * RT;
            if (which == 2) stat = __int_as_float(r < u.rows ? limit_of_row(a, u, r) : 0);
            else stat = r < u.rows ? (which == 0 ? a.lse[stats + r] : -a.delta[stats + r]) : (which == 0 ? INFINITY : 0.f);
        }
    };
    if constexpr (WHOLE) {
        // (of a whole tile: no row is behind the last)
#pragma unroll
        for (int i = 0; i < QG::PER; i++) {
            const int row = QG::row_of(i), pos = fdiv(row, a.by_group), d = QG::column_of(i, a.D);
            const unsigned at = pos, head = row - pos * a.group;
            qoff[i] = (at * (unsigned)a.qs[0] + head * (unsigned)a.qs[1] + d) * (unsigned)sizeof(T);
            goff[i] = (at * (unsigned)a.gs[0] + head * (unsigned)a.gs[1] + d) * (unsigned)sizeof(T);
        }
    }
    if (t < t1) request(t);
    const T *kb = reinterpret_cast<const T *>(a.k) + (long)u.k0 * a.ks[0] + u.h * a.ks[1], *vb = reinterpret_cast<const T *>(a.v) + (long)u.k0 * a.vs[0] + u.h * a.vs[1];
    Frag<P> k[NK], v[Shape::V_LDS ? 1 : NK];
    unsigned char *s_v = lds + BUFFERS * Shape::BYTES;
    if constexpr (Shape::V_LDS) {
        typename Shape::V tile;
        tile.load(a.D, [&](int i) INLINE { return vb + (long)min(key0 + i, u.lk - 1) * a.vs[0]; });
        tile.template store<false>(s_v, a.D);      // (a key behind the last: a column of its own, which is not stored)
    }
    {
        const long at = min(key, u.lk - 1);
        const T *kr = kb + at * a.ks[0], *vr = vb + at * a.vs[0];
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
    int buffer = 0, masked_rows = 0;

    for (; t < t1; t++) {
        unsigned char *s_q = lds + (BUFFERS == 2 ? buffer * Shape::BYTES : 0), *s_g = s_q + QG::BYTES;
        float *s_lse = reinterpret_cast<float *>(s_q + 2 * QG::BYTES), *s_delta = s_lse + RT;
        const int *s_lim = reinterpret_cast<const int *>(s_delta + RT);
        // (a row that does not read all of the tile's keys, or reads one key alone)
        const int least = limit_of_row(a, u, t * RT);
        const bool masked = least < keys_end || least <= 1;
        if constexpr (BUFFERS == 1) __syncthreads();
        if (t * RT + RT > u.rows) g.zero_rows([&](int i) INLINE { return t * RT + i >= u.rows; });
        if (masked) {
            const bool bad = __any(not_finite<T>(q) || not_finite<T>(g));
            if (lane == 0) s_bad[buffer][wave] = bad;
        }
        q.template store<false>(s_q, a.D);
        g.template store<false>(s_g, a.D);
        if (threadIdx.x < 3 * RT) s_lse[threadIdx.x] = stat;
        __syncthreads();
        if (t + 1 < t1) request(t + 1);
        const bool bad = masked && (s_bad[buffer][0] | s_bad[buffer][1] | s_bad[buffer][2] | s_bad[buffer][3]);
        if (bad) masked_rows = (t + 1) * RT;
        buffer ^= 1;
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
            if (masked) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int4 lm = *reinterpret_cast<const int4 *>(s_lim + i * 32 + j * 8 + half * 4);
                    const int lr[4] = {lm.x, lm.y, lm.z, lm.w};
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const bool read = key < lr[r];
                        p[j * 4 + r] = read ? p[j * 4 + r] : 0.f;
                        ds[j * 4 + r] = read ? (lr[r] == 1 ? ds[j * 4 + r] * 0.f : ds[j * 4 + r]) : 0.f;
                    }
                }
            }
            if (bad) {
                __syncthreads();
                clean_rows<QG>(s_q, i * 32);
                clean_rows<QG>(s_g, i * 32);
                __syncthreads();
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
    if (masked_rows > 0) {      // (rows of the tiles that were cleaned)
        const int first_row = t0 * RT, end = min(masked_rows, u.rows);
        auto read = [&](int j) INLINE { return key < limit_of_row(a, u, j); };
        take_in<T, false>(dv, a.D, first_row, end, [&](int j) INLINE { return row_at<T>(a.g, a.gs, a, u, j); }, read);
        take_in<T, true>(dk, a.D, first_row, end, [&](int j) INLINE { return row_at<T>(a.q, a.qs, a, u, j); }, read);
    }
    if (!live) return;
    const float fk = walk.splits > 1 ? 1.f : a.scale;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + j * 8 + half * 4;
            const float x[4] = {dk[i][j * 4] * fk, dk[i][j * 4 + 1] * fk, dk[i][j * 4 + 2] * fk, dk[i][j * 4 + 3] * fk};
            const float y[4] = {dv[i][j * 4], dv[i][j * 4 + 1], dv[i][j * 4 + 2], dv[i][j * 4 + 3]};
            if (walk.splits > 1) {
                const long step = (long)a.tiles * a.Hkv * kRows, line = ((long)u.at * a.Hkv + u.h) * kRows + tile_key;
                store4<float>(a.part + (2L * u.split * step + line) * part_width(a.D) + d, x, a.D - d);
                store4<float>(a.part + ((2L * u.split + 1) * step + line) * part_width(a.D) + d, y, a.D - d);
            } else {
                const long at = ((long)(u.k0 + key) * a.Hkv + u.h) * a.D + d;
                if (a.gk) store4<T>(reinterpret_cast<T *>(a.gk) + at, x, a.D - d);
                if (a.gv) store4<T>(reinterpret_cast<T *>(a.gv) + at, y, a.D - d);
            }
        }
}

template <typename T, int DP, int NP, bool WHOLE> __global__ void __launch_bounds__(256, (KvShape<T, DP, WHOLE>::WAVES)) packed_bwd_kv_kernel(PackedArgs a)
{
    const PackedUnit u = unit_of<true>(a, blockIdx.x);
    if (u.tile * kRows >= u.lk) return;
    constexpr int TERMS = kWeightTerms<T, WHOLE>;
    with_terms<TERMS>(a, u, TERMS == 1 && few_rows(a, u), [](const PackedArgs &b, const PackedUnit &w, auto terms) INLINE { bwd_keys<T, DP, NP, WHOLE, decltype(terms)::value>(b, w); });
}

// Sums of the workgroups that shared a walk: a workgroup to 16 rows (or keys) of a tile, a thread to four columns and those 64 further on, four splits requested at a time.
template <typename T, bool KV> __global__ void __launch_bounds__(256) packed_bwd_join_kernel(PackedArgs a)
{
    const PackedUnit u = unit_of<KV>(a, blockIdx.x / 8);
    const int line = blockIdx.x % 8 * 16 + threadIdx.x / 16, at = u.tile * kRows + line, which = KV ? blockIdx.y : 0;
    const int splits = (KV ? key_walk(a, u) : row_walk(a, u)).splits;
    if (splits == 1 || at >= (KV ? u.lk : u.rows) || (KV && !(which ? a.gv : a.gk))) return;
    const long step = (long)a.tiles * a.Hkv * kRows, first = ((long)u.at * a.Hkv + u.h) * kRows + line;
    const int width = part_width(a.D);
    T *to;
    if constexpr (KV) to = reinterpret_cast<T *>(which ? a.gv : a.gk) + ((long)(u.k0 + at) * a.Hkv + u.h) * a.D;
    else to = const_cast<T *>(row_at<T>(a.gq, a.gs, a, u, at));
    const float f = which == 0 ? a.scale : 1.f;
    for (int d = threadIdx.x % 16 * 4; d < a.D; d += 64) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < splits; s0 += 4) {
            float4 y[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                y[i] = *reinterpret_cast<const float4 *>(a.part + (((long)min(s0 + i, splits - 1) * (KV ? 2 : 1) + which) * step + first) * width + d);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (s0 + i >= splits) continue;
                x[0] += y[i].x; x[1] += y[i].y; x[2] += y[i].z; x[3] += y[i].w;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] *= f;
        store4<T>(to + d, x, a.D - d);
    }
}

// delta alone, where the queries' gradient is not wanted: one wavefront to a row (and to the rows a launch's wavefronts further on)
constexpr long kDeltaBlocks = 1L << 20;
template <typename T> __global__ void __launch_bounds__(256) packed_delta_kernel(PackedArgs a)
{
    const long rows = (long)a.T * a.group, total = rows * a.Hkv;
    const int lane = threadIdx.x & 63;
    for (long at = (long)blockIdx.x * 4 + (threadIdx.x >> 6); at < total; at += 4L * gridDim.x) {
        const int h = (int)(at / rows), row = (int)(at - h * rows), pos = fdiv(row, a.by_group);
        const long from = (long)pos * a.gs[0] + (long)(h * a.group + row - pos * a.group) * a.gs[1];
        const T *g = reinterpret_cast<const T *>(a.g) + from, *o = reinterpret_cast<const T *>(a.o) + from;
        const T *low = a.o_low ? reinterpret_cast<const T *>(a.o_low) + from : nullptr;
        float x = 0.f;
        for (int d = lane; d < a.D; d += 64) x = fmaf(elem_to_f32<T>(g[d]), elem_to_f32<T>(o[d]) + (low ? elem_to_f32<T>(low[d]) : 0.f), x);
        x = lanes_sum<64>(x);
        if (lane == 0) a.delta[at] = x;
    }
}

struct BwdPlan { int q_tiles, kv_tiles; Split q, kv; size_t delta_bytes, bytes; };
template <typename T> BwdPlan bwd_plan(const d2c_packed_attention_desc &q)
{
    BwdPlan p{};
    const long group = q.Hq / q.Hkv, rows = q.queries * group, cus = std::max(d2c_num_cus(), 1);
    p.q_tiles = tiles_of(rows, q.sequences);
    p.kv_tiles = tiles_of(q.keys, q.sequences);
    const double unit = kRows * (part_width(q.D) * 4.0);
    pick_width(q.D, fast_kernels(q, true), [&](auto width, auto whole) {
        constexpr int DP = decltype(width)::DP, NP = decltype(width)::NP;
        constexpr bool WHOLE = decltype(whole)::value;
        using Q = QShape<T, DP, WHOLE>;
        using KV = KvShape<T, DP, WHOLE>;
        p.q = split_walks(q, (long)p.q_tiles * q.Hkv, cus * resident(reinterpret_cast<const void *>(&packed_bwd_q_kernel<T, DP, NP, WHOLE>), Q::LDS), q.keys, Q::KT, unit);
        p.kv = split_walks(q, (long)p.kv_tiles * q.Hkv, cus * resident(reinterpret_cast<const void *>(&packed_bwd_kv_kernel<T, DP, NP, WHOLE>), KV::LDS), rows, KV::RT, 2 * unit);
        return 0;
    });
    p.delta_bytes = d2c_align_up((size_t)rows * q.Hkv * 4);
    const size_t q_part = p.q.splits > 1 ? (size_t)p.q.splits * p.q_tiles * q.Hkv * (size_t)unit : 0, kv_part = p.kv.splits > 1 ? 2 * (size_t)p.kv.splits * p.kv_tiles * q.Hkv * (size_t)unit : 0;
    p.bytes = p.delta_bytes + d2c_align_up(std::max(q_part, kv_part));
    return p;
}

template <typename T, int DP, int NP, bool WHOLE> int launch_bwd(PackedArgs a, const BwdPlan &p, hipStream_t st)
{
    if (a.T > 0 && !a.gq && (a.gk || a.gv)) {
        hipLaunchKernelGGL(packed_delta_kernel<T>, dim3((unsigned)std::min(((long)a.T * a.Hq + 3) / 4, kDeltaBlocks)), dim3(256), 0, st, a);
        if (int rc = d2c_check_launch("packed_delta_kernel")) return rc;
    } else if (a.T > 0 && a.gq) {
        constexpr int lds = QShape<T, DP, WHOLE>::LDS;
        if (int rc = d2c_allow_lds(reinterpret_cast<const void *>(&packed_bwd_q_kernel<T, DP, NP, WHOLE>), lds, "packed_bwd_q_kernel")) return rc;
        a.tiles = p.q_tiles; a.splits = p.q.splits; a.chunk = p.q.chunk; a.step = QShape<T, DP, WHOLE>::KT;
        hipLaunchKernelGGL((packed_bwd_q_kernel<T, DP, NP, WHOLE>), dim3((unsigned)(a.tiles * a.Hkv * a.splits)), dim3(256), lds, st, a);
        if (int rc = d2c_check_launch("packed_bwd_q_kernel")) return rc;
        if (a.splits > 1) {
            hipLaunchKernelGGL((packed_bwd_join_kernel<T, false>), dim3((unsigned)(a.tiles * a.Hkv * 8)), dim3(256), 0, st, a);
            if (int rc = d2c_check_launch("packed_bwd_join_kernel")) return rc;
        }
    }
    if (a.Tk == 0 || !(a.gk || a.gv)) return D2C_OK;
    constexpr int lds = KvShape<T, DP, WHOLE>::LDS;
    if (int rc = d2c_allow_lds(reinterpret_cast<const void *>(&packed_bwd_kv_kernel<T, DP, NP, WHOLE>), lds, "packed_bwd_kv_kernel")) return rc;
    a.tiles = p.kv_tiles; a.splits = p.kv.splits; a.chunk = p.kv.chunk; a.step = KvShape<T, DP, WHOLE>::RT;
    hipLaunchKernelGGL((packed_bwd_kv_kernel<T, DP, NP, WHOLE>), dim3((unsigned)(a.tiles * a.Hkv * a.splits)), dim3(256), lds, st, a);
    if (int rc = d2c_check_launch("packed_bwd_kv_kernel")) return rc;
    if (a.splits == 1) return D2C_OK;
    hipLaunchKernelGGL((packed_bwd_join_kernel<T, true>), dim3((unsigned)(a.tiles * a.Hkv * 8), 2), dim3(256), 0, st, a);
    return d2c_check_launch("packed_bwd_join_kernel");
}
template <typename T> int backward(PackedArgs a, const d2c_packed_attention_desc &q, void *ws, size_t ws_bytes, hipStream_t st)
{
    const BwdPlan p = bwd_plan<T>(q);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 255u))) {
        d2c_set_error("workspace of %zu bytes (256-byte aligned) required, got %zu at %p", p.bytes, ws_bytes, ws);
        return D2C_ERR_WORKSPACE;
    }
    a.delta = (float *)ws; a.part = (float *)((char *)ws + p.delta_bytes);
    return pick_width(q.D, fast_kernels(q, true), [&](auto width, auto whole) { return launch_bwd<T, decltype(width)::DP, decltype(width)::NP, decltype(whole)::value>(a, p, st); });
}

}  // namespace

extern "C" size_t d2c_packed_attention_backward_workspace_bytes(const d2c_packed_attention_desc *q)
{
    if (d2c_packed_attention_check(q) != D2C_OK || (q->queries == 0 && q->keys == 0)) return 0;
    return q->dtype == D2C_BF16 ? bwd_plan<bf16_t>(*q).bytes : bwd_plan<float>(*q).bytes;
}

extern "C" int d2c_packed_attention_backward(const d2c_packed_attention_desc *q, const void *grad_out, const void *query, const void *key,
                                             const void *value, const int32_t *starts, const int32_t *key_starts, const void *out,
                                             const void *out_low, const float *lse, void *grad_query, void *grad_key, void *grad_value,
                                             void *ws, size_t ws_bytes, void *stream)
{
    if (int rc = d2c_packed_attention_check(q)) return rc;
    if (q->queries == 0 && q->keys == 0) return D2C_OK;
    if ((q->queries > 0 && (!grad_out || !query || !out || !lse)) || (q->keys > 0 && (!key || !value)) || !starts) {
        d2c_set_error("null tensor pointer");
        return D2C_ERR_SHAPE;
    }
    PackedArgs a = make_args(*q, starts, key_starts);
    a.g = grad_out; a.q = query; a.k = key; a.v = value; a.o = out;
    a.o_low = q->dtype == D2C_BF16 ? out_low : nullptr;
    a.lse = const_cast<float *>(lse);
    a.gq = grad_query; a.gk = grad_key; a.gv = grad_value;
    return q->dtype == D2C_BF16 ? backward<bf16_t>(a, *q, ws, ws_bytes, (hipStream_t)stream) : backward<float>(a, *q, ws, ws_bytes, (hipStream_t)stream);
}
