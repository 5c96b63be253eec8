// Attention of one map's positions to those of another: forward pass.  Formulas and operand orders: d2c_attention.hpp.
//
// A workgroup takes one key head, 128 rows (32 to a wavefront) and walks over the keys a tile at a time, K and V through LDS, the
// next tile requested while this one is worked on.  Few rows: the wavefronts share them and split the keys of a tile, and several workgroups share the keys;
// their results are joined by attn_join_kernel.
// Up to 8 rows of a key head run on attn_token_kernel, where no matrix instruction has columns to fill.
#include <mutex>
#include <type_traits>
#include "d2c_attention.hpp"

using namespace d2c_attn;

namespace {

// The keys of a tile of KT that are to be read: bit i of word j is key k0 + 64 j + i.  Requested as bytes two tiles ahead.
template <int KT> struct KeyBits {
    static constexpr int WORDS = (KT + 63) / 64;
    bool b[WORDS];
    D2C_DEV void request(const Args &a, int n, int keys, int k0)
    {
#pragma unroll
        for (int j = 0; j < WORDS; j++) {
            const int i = j * 64 + (int)(threadIdx.x & 63), key = k0 + i;
            b[j] = i < KT && key < keys && (!a.mask || a.mask[(long)n * a.Lk + key]);
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
    // wavefronts to a SIMD: one where three terms of wide rows and the sums of split keys do not fit half of the registers (20 rows of 8 heads of 128 reading
    // 30000: 158 us spilled, 87.5 so; whole tiles of rows spill less, and one to a SIMD takes longer: 2048 reading 4096 227 us, 265)
    static constexpr int WAVES = sizeof(T) == 4 && DP == 128 && WK > 1 ? 1 : 2;
    static constexpr int JOIN = WK > 1 ? 4 * 32 * (DP + 2) * 4 : 0;
    // two tiles of each where three workgroups of a compute unit have room for them: one barrier a tile
    static constexpr int BUFFERS = 4 * KV::BYTES <= 52 << 10 ? 2 : 1;
    static constexpr int LDS = 2 * BUFFERS * KV::BYTES > JOIN ? 2 * BUFFERS * KV::BYTES : JOIN;
};

// WK: wavefronts that share rows and split the keys of a tile.
//
// One pass over the keys with the running maximum and sum of a softmax; the weights p go from one product's accumulator into the next one's operand without
// leaving their registers, so that LDS holds K and V alone, which come through it once for 128 rows.  Registers are kept to what three workgroups of a compute
// unit have room for at 64 channels (two take 1.18 times as long, one 1.95).  Bound: the matrix instructions (busy 0.41 of the time at 64 channels, 0.43 at 128)
// and the exponentials, maxima, sums and roundings between them (0.66, 0.35), which do not overlap further at the clock that the card keeps under them (1.95 GHz): without the
// exponentials 0.80 of the time, without the second product 0.80, without either's loads 0.95 each.
// Measured, bfloat16: 12960 positions reading 25920, 8 heads of 64, 0.82 ms (0.84 PFLOP/s; a library product of 8192 cubed 1.27); 1620 reading 64800, 8 heads of
// 128 that share 2 key heads, 0.46 ms with the join (0.94 PFLOP/s).  float32: 1417 reading 3001, 6 heads of 40, 43 us.
template <typename T, int DP, int NP, int WK, bool WHOLE> __global__ void __launch_bounds__(256, (FwdShape<T, DP, WK, WHOLE>::WAVES)) attn_fwd_kernel(Args a)
{
    using Shape = FwdShape<T, DP, WK, WHOLE>;
    using KV = typename Shape::KV;
    constexpr int P = kTerms<T>, PW = kWeightTerms<T, WHOLE>, ND = DP / 32, NK = kSteps<NP>, KW = Shape::KW, KT = Shape::KT, NS = KW / 32, WORDS = KeyBits<KT>::WORDS;
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int BUFFERS = Shape::BUFFERS;
    constexpr bool END = WHOLE && NP % 2 == 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, wk = wave % WK;
    const Unit unit = unit_of(a);
    const Head hd = unit.head;
    const int tile_row = (wave / WK) * 32 + (lane & 31), row = unit.tile * Shape::ROWS + tile_row;
    const int keys = keys_of(a, hd.n), tiles = (keys + KT - 1) / KT;
    const int t1 = (int)((long)tiles * (unit.split + 1) / unit.splits);
    int t = (int)((long)tiles * unit.split / unit.splits);

    KV k, v;
    const KeyTiles<T, KV, KT, WORDS, WHOLE> source(a, hd);
    KeyBits<KT> bits;
    uint64_t next[WORDS];
    auto request = [&](int tile) INLINE { source.request(a, k, v, tile, next); };
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
            const Raw8<T> raw = load8_of<WHOLE, T>(qr, d, a.D, row < a.rows);
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
    // (float32 has its scale in the rows already: the largest score's weight is 1 to the last bit, and a row with one key takes its value as it is)
    const float c = sizeof(T) == 4 ? 1.f : a.scale2;
    int buffer = 0;

    for (; t < t1; t++) {
        uint64_t now[WORDS];
#pragma unroll
        for (int j = 0; j < WORDS; j++) now[j] = next[j];
        // (with two buffers: who writes one has passed the barrier behind which the other was read, so nobody reads this one any more)
        unsigned char *s_k = lds + (BUFFERS == 2 ? buffer * 2 * KV::BYTES : 0), *s_v = s_k + KV::BYTES;
        buffer ^= 1;
        if constexpr (BUFFERS == 1) __syncthreads();
        if (!all_keys<KT>(now)) v.zero_rows([&](int i) INLINE { return !has_key(now, i); });
        k.template store<END>(s_k, a.D);
        v.template store<false>(s_v, a.D);      // (its piece behind the end makes columns of o that are not stored)
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
            for (int ks = 0; ks < NK; ks++) mma(s[i], KV::rows(s_k, wk * KW + i * 32 + (lane & 31), ks, half), q[ks]);
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
                const Frag<PW> pf = make_frag<PW, WEIGHTS>(p + kk * 8);
#pragma unroll
                for (int d = 0; d < ND; d++) mma(o[d], KV::columns(s_v, wk * KW + i * 32 + kk * 16, d * 32, lane), pf);
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
    if (unit.splits > 1) {
        const long at = ((long)unit.split * a.shared + unit.part) * Shape::ROWS + tile_row;
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
    const int pos = row / a.group, head = hd.h * a.group + row - pos * a.group;
    T *orow = reinterpret_cast<T *>(a.out) + (((long)hd.n * a.Lq + pos) * a.Hq + head) * a.D;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + j * 8 + half * 4;
            const float x[4] = {o[i][j * 4] * inv, o[i][j * 4 + 1] * inv, o[i][j * 4 + 2] * inv, o[i][j * 4 + 3] * inv};
            store4<T>(orow + d, x, a.D - d);
            if (a.out_low) store4_low<T>(reinterpret_cast<T *>(a.out_low) + (orow - reinterpret_cast<T *>(a.out)) + d, x, a.D - d);
        }
    if (a.lse && half == 0) a.lse[hd.nh * a.rows + row] = l == 0.f ? INFINITY : mc + log2f(l);
}

template <int LANES, typename Op> D2C_DEV float over_groups(float v, Op op)      // over the lanes that lie a multiple of LANES apart
{
    if constexpr (LANES <= 4) v = op(v, dpp_f32<0x124>(v));    // lanes of sixteen, turned by 4
    if constexpr (LANES <= 8) v = op(v, dpp_f32<0x128>(v));    // ... by 8
    if constexpr (LANES <= 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    float x, y;
    other_half(v, x, y);
    return op(x, y);
}

// x + the products of two pairs
D2C_DEV float dot_pair(uint32_t a, uint32_t b, float x)
{
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, a), __builtin_bit_cast(bf16x2_t, b), x, false);
}
// 16 bytes against 16 bytes
template <typename T> D2C_DEV float dot_words(const uint4 &a, const uint4 &b)
{
    if constexpr (sizeof(T) == 2) return dot_pair(a.w, b.w, dot_pair(a.z, b.z, dot_pair(a.y, b.y, dot_pair(a.x, b.x, 0.f))));
    else return fmaf(__uint_as_float(a.w), __uint_as_float(b.w), fmaf(__uint_as_float(a.z), __uint_as_float(b.z),
                fmaf(__uint_as_float(a.y), __uint_as_float(b.y), __uint_as_float(a.x) * __uint_as_float(b.x))));
}

template <typename T, int LANES, int R> struct TokenShape {
    static constexpr int VEC = 16 / (int)sizeof(T), DP = LANES * VEC, LOADS = R <= 4 ? 4 : 2, KEYS = 64 / LANES, STEP = 4 * LOADS * KEYS;
};

// One to eight rows (a token, or a few that share a key head): no matrix instructions, whose 32 columns would be empty, but one pass over the memory by
// lanes.  LANES lanes hold a key's row, 16 bytes each, so that a load of the wavefront takes 64 / LANES whole rows; scores are summed over these lanes, and
// every group of lanes keeps its own maximum, sum and output of each of the R rows until the end.  No LDS and no barrier on the way, the next keys requested
// while these are worked on.  Bound: memory, latency where the memory is short.  Measured with the join: one token of 16 heads that share 4, 12960
// positions of 64 channels, bfloat16, 12.4 us (13 MB: 2.6 at a copy's rate; two launches are 8 of them); two samples' 30000 positions of 128 channels 22.4 us,
// float32 23 (attn_fwd_kernel 28.8 and 58).  Weights stay in float32: bfloat16 pairs on the dot instruction took 48.0, 48.1 us (one row), 21.0, 21.6 (four), 68.5, 71.6
// (eight rows of 16 heads on 30000 positions of 128 channels) and lost 2^-9 of each.
template <typename T, int LANES, int R, bool WHOLE> __global__ void __launch_bounds__(256) attn_token_kernel(Args a)
{
    using Shape = TokenShape<T, LANES, R>;
    constexpr int VEC = Shape::VEC, DP = Shape::DP, LOADS = Shape::LOADS, KEYS = Shape::KEYS, STEP = Shape::STEP;
    __shared__ __align__(16) float s_o[4][R][DP];
    __shared__ float2 s_ml[4][R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d0 = lane % LANES * VEC;
    const Unit unit = unit_of(a);
    const Head hd = unit.head;
    const int keys = keys_of(a, hd.n), steps = (keys + STEP - 1) / STEP;
    const int t1 = (int)((long)steps * (unit.split + 1) / unit.splits);
    int t = (int)((long)steps * unit.split / unit.splits);
    const T *kb = reinterpret_cast<const T *>(a.k) + hd.n * a.ks[0] + hd.h * a.ks[2];
    const T *vb = reinterpret_cast<const T *>(a.v) + hd.n * a.vs[0] + hd.h * a.vs[2];

    auto load = [&](const T *row) INLINE {      // this lane's 16 bytes; zeros behind the row's end
        if constexpr (WHOLE) {
            const AnyVec<T> v = load_any(row + min(d0, a.D - VEC));
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else return d0 < a.D ? load_run<T>(row + d0, a.D - d0) : make_uint4(0, 0, 0, 0);
    };
    uint4 k[LOADS], v[LOADS];
    bool there[LOADS];
    auto request = [&](int step) INLINE {
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            const int key = step * STEP + (u * 4 + wave) * KEYS + lane / LANES;
            const long at = min(key, keys - 1);
            there[u] = key < keys && (!a.mask || a.mask[(long)hd.n * a.Lk + at]);
            k[u] = load(kb + at * a.ks[1]);
            v[u] = load(vb + at * a.vs[1]);
        }
    };
    if (t < t1) request(t);
    uint4 q[R];
    float o[R][VEC], m[R], l[R];      // (m: of the scores in units of scale * log2(e))
#pragma unroll
    for (int r = 0; r < R; r++) {
        const uint4 w = load(row_at<T>(a.q, a.qs, a, hd, min(r, a.rows - 1)));
        q[r] = r < a.rows ? w : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < VEC; i++) o[r][i] = 0.f;
        m[r] = -INFINITY;
        l[r] = 0.f;
    }
    for (; t < t1; t++) {
        uint4 vw[LOADS];
        float s[LOADS][R];
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            vw[u] = there[u] ? v[u] : make_uint4(0, 0, 0, 0);
            // (a lane behind a row's end has its last piece again, which is no part of the score)
            uint4 kw = k[u];
            if (WHOLE && a.D < DP && d0 >= a.D) kw = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float x = lanes_sum<LANES>(dot_words<T>(q[r], kw)) * a.scale2;
                s[u][r] = there[u] ? x : -INFINITY;
            }
        }
        if (t + 1 < t1) request(t + 1);
#pragma unroll
        for (int r = 0; r < R; r++) {
            float top = s[0][r];
#pragma unroll
            for (int u = 1; u < LOADS; u++) top = fmaxf(top, s[u][r]);
            // (the maximum follows where it has grown by more than 8, as in attn_fwd_kernel)
            if (__any(top > m[r] + 8.f)) {
                const float grown = fmaxf(top, m[r]), f = grown == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - grown);
                m[r] = grown;
                l[r] *= f;
#pragma unroll
                for (int i = 0; i < VEC; i++) o[r][i] *= f;
            }
            const float base = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - base);
                l[r] += s[u][r];
            }
        }
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            alignas(16) T e[VEC];
            float vf[VEC];
            *reinterpret_cast<uint4 *>(e) = vw[u];
#pragma unroll
            for (int i = 0; i < VEC; i++) vf[i] = elem_to_f32<T>(e[i]);
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < VEC; i++) o[r][i] = fmaf(s[u][r], vf[i], o[r][i]);
        }
    }
    // the groups of a wavefront, two values to a step where half the wavefront can go on with either (32 sums of 8 lanes: 56 instructions for 256), then the
    // wavefronts
    float x[R * VEC];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const float top = over_groups<LANES>(m[r], [](float x, float y) INLINE { return fmaxf(x, y); });
        const float f = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - top);
        l[r] = over_groups<LANES>(l[r] * f, [](float x, float y) INLINE { return x + y; });
#pragma unroll
        for (int i = 0; i < VEC; i++) x[r * VEC + i] = o[r][i] * f;
        if (lane == 0) s_ml[wave][r] = make_float2(top, l[r]);
    }
    constexpr int HALVINGS = LANES <= 16 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < R * VEC / 2; i++) {
        const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]), false, false);
        x[i] = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    }
    if constexpr (HALVINGS == 2) {
#pragma unroll
        for (int i = 0; i < R * VEC / 4; i++) {
            const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]), false, false);
            x[i] = __uint_as_float(w[0]) + __uint_as_float(w[1]);
        }
    }
#pragma unroll
    for (int i = 0; i < (R * VEC >> HALVINGS); i++) {
        if constexpr (LANES <= 4) x[i] += dpp_f32<0x124>(x[i]);
        if constexpr (LANES <= 8) x[i] += dpp_f32<0x128>(x[i]);
        const int at = HALVINGS == 2 ? 4 * i + (lane >> 4 & 1) * 2 + (lane >> 5) : 2 * i + (lane >> 5);
        if (LANES >= 16 || (lane & 15) < LANES) s_o[wave][at / VEC][d0 + at % VEC] = x[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(R, a.rows) * DP; i += 256) {
        const int r = i / DP, d = i - r * DP;
        if (d >= a.D) continue;
        float top = s_ml[0][r].x, sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 1; w < 4; w++) top = fmaxf(top, s_ml[w][r].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = __builtin_amdgcn_exp2f(s_ml[w][r].x - base);
            sum = fmaf(s_ml[w][r].y, f, sum);
            x = fmaf(s_o[w][r][d], f, x);
        }
        if (unit.splits > 1) {
            const long at = ((long)unit.split * a.shared + unit.part) * R + r;
            a.part[at * part_width(a.D) + d] = x;
            if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + at * 2) = make_float2(top, sum);
        } else {
            const float y = sum == 0.f ? 0.f : x / sum;
            const T rounded = f32_to_elem<T>(y);
            const_cast<T *>(row_at<T>(a.out, a.gs, a, hd, r))[d] = rounded;
            if (a.out_low) const_cast<T *>(row_at<T>(a.out_low, a.gs, a, hd, r))[d] = f32_to_elem<T>(y - elem_to_f32<T>(rounded));
            if (a.lse && d == 0) a.lse[hd.nh * a.rows + r] = sum == 0.f ? INFINITY : top + log2f(sum);
        }
    }
}

// The partial results of `splits` workgroups.  LANES lanes take four of a row's columns each, `groups` (a power of two) of them the splits in turn, four
// requested at a time (eight are no quicker); their sums meet in LDS.  Latency counts: 16 rows of 102 splits 13.6 us as a wavefront each that walks over them, 4.6
// as here; 26624 rows of 7 splits of 64 columns 11.5 us (4.1 TB/s of the 48 MB), 22 with as many groups as there are splits for.
template <typename T, int LANES> __global__ void __launch_bounds__(256) attn_join_kernel(Args a, int groups, int tile_rows)
{
    __shared__ float4 s_x[256];
    __shared__ float2 s_ml[256];
    const int per = 256 / (LANES * groups), lane = threadIdx.x % LANES, group = threadIdx.x / LANES % groups;
    const int total = a.shared * tile_rows, at = (int)blockIdx.x * per + threadIdx.x / (LANES * groups);
    const int part = at / tile_rows, unit = a.whole + part, heads = a.N * a.Hkv, tile = unit / heads, nh = unit - tile * heads;
    const int row = tile * tile_rows + at - part * tile_rows;
    const bool live = at < total && row < a.rows;
    const int d = lane * 4;
    float all = -INFINITY, l = 0.f;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
        for (int s0 = group; s0 < a.splits; s0 += 4 * groups) {
            float2 ml[4];
            float4 y[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const long from = (long)min(s0 + u * groups, a.splits - 1) * total + at;
                ml[u] = *reinterpret_cast<const float2 *>(a.part_ml + from * 2);
                y[u] = *reinterpret_cast<const float4 *>(a.part + from * part_width(a.D) + min(d, part_width(a.D) - 4));
            }
            float top = all;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (s0 + u * groups >= a.splits) ml[u] = make_float2(-INFINITY, 0.f);
                top = fmaxf(top, ml[u].x);
            }
            const float base = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f(all - base);
            all = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] *= f;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (s0 + u * groups >= a.splits) continue;
                const float g = __builtin_amdgcn_exp2f(ml[u].x - base);
                l = fmaf(ml[u].y, g, l);
                x[0] = fmaf(y[u].x, g, x[0]); x[1] = fmaf(y[u].y, g, x[1]); x[2] = fmaf(y[u].z, g, x[2]); x[3] = fmaf(y[u].w, g, x[3]);
            }
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
    const int n = nh / a.Hkv, pos = row / a.group, head = (nh - n * a.Hkv) * a.group + row - pos * a.group;
    T *orow = reinterpret_cast<T *>(a.out) + (((long)n * a.Lq + pos) * a.Hq + head) * a.D;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] *= inv;
    if (d < a.D) {
        store4<T>(orow + d, x, a.D - d);
        if (a.out_low) store4_low<T>(reinterpret_cast<T *>(a.out_low) + (orow - reinterpret_cast<T *>(a.out)) + d, x, a.D - d);
    }
    if (a.lse && lane == 0) a.lse[(long)nh * a.rows + row] = l == 0.f ? INFINITY : top + log2f(l);
}

// f(Width, WK, WHOLE) as constants
template <typename T, typename F> auto for_shape(const d2c_attention_desc &q, bool few, F f)
{
    constexpr int WK = sizeof(T) == 2 ? 4 : 2;
    return for_width<T, false>(q, [&](auto width, auto whole) {
        return few ? f(width, std::integral_constant<int, WK>{}, whole) : f(width, std::integral_constant<int, 1>{}, whole);
    });
}

// f(LANES, R, WHOLE) of attn_token_kernel as constants
template <typename T, typename F> auto for_token(const d2c_attention_desc &q, long rows, F f)
{
    const int D = q.D;
    auto with_rows = [&](auto lanes, auto whole) {
        if (rows <= 1) return f(lanes, std::integral_constant<int, 1>{}, whole);
        if (rows <= 2) return f(lanes, std::integral_constant<int, 2>{}, whole);
        if (rows <= 4) return f(lanes, std::integral_constant<int, 4>{}, whole);
        return f(lanes, std::integral_constant<int, 8>{}, whole);
    };
    auto pick = [&](auto lanes) { return fast_kernels(q, false) ? with_rows(lanes, std::true_type{}) : with_rows(lanes, std::false_type{}); };
    constexpr int L32 = 32 * (int)sizeof(T) / 16;
    if (D <= 32) return pick(std::integral_constant<int, L32>{});
    if (D <= 64) return pick(std::integral_constant<int, 2 * L32>{});
    return pick(std::integral_constant<int, 4 * L32>{});
}

// What a call runs on: up to 8 rows on attn_token_kernel; up to 32 are shared by the wavefronts of a workgroup, which split the keys of a tile (WK > 1)
struct FwdPlan { bool token, few; int tile_rows; Walks walks; size_t part_bytes, bytes; };
template <typename T> FwdPlan fwd_plan(const d2c_attention_desc &q)
{
    FwdPlan p;
    const long rows = (long)q.Lq * (q.Hq / q.Hkv), heads = (long)q.N * q.Hkv;
    p.token = rows <= 8;
    p.few = rows <= 32;
    if (p.token) for_token<T>(q, rows, [&](auto lanes, auto r, auto whole) {
        constexpr int LANES = decltype(lanes)::value, R = decltype(r)::value;
        using Shape = TokenShape<T, LANES, R>;
        p.tile_rows = R;
        const long places = 2L * std::max(d2c_num_cus(), 1);
        // (a step's bytes, from every place, at 5 TB/s)
        p.walks = plan_walks(heads, (q.Lk + Shape::STEP - 1) / Shape::STEP, places, 2.0 * Shape::STEP * q.D * sizeof(T) * places / 5e6, (double)R * (part_width(q.D) * 4 + 8),
                             part_limit(q));
        return 0;
    });
    else for_shape<T>(q, p.few, [&](auto width, auto wk, auto whole) {
        constexpr int DP = decltype(width)::DP, NP = decltype(width)::NP, WK = decltype(wk)::value;
        constexpr bool WHOLE = decltype(whole)::value;
        using Shape = FwdShape<T, DP, WK, WHOLE>;
        p.tile_rows = Shape::ROWS;
        const long units = heads * ((rows + Shape::ROWS - 1) / Shape::ROWS), steps = (q.Lk + Shape::KT - 1) / Shape::KT;
        const long places = (long)std::max(d2c_num_cus(), 1) *
            resident(reinterpret_cast<const void *>(&attn_fwd_kernel<T, DP, NP, WK, WHOLE>), Shape::LDS);
        // (a step: 64 keys of 64 channels take 2 us with every place taken, float32's six products three times as long)
        p.walks = plan_walks(units, steps, places, 2.0 * Shape::KT / 64 * DP / 64 * (sizeof(T) == 2 ? 1 : 3) / WK, (double)Shape::ROWS * (part_width(q.D) * 4 + 8), part_limit(q));
        return 0;
    });
    const size_t lines = (size_t)p.walks.splits * p.walks.shared * p.tile_rows;
    p.part_bytes = d2c_align_up(lines * part_width(q.D) * 4);
    p.bytes = p.part_bytes + d2c_align_up(lines * 8);
    return p;
}

template <typename T, int LANES> int launch_join(const Args &a, int tile_rows, hipStream_t st)
{
    // (more lanes to a row only while all of them have a place at once)
    const long total = (long)a.shared * tile_rows, places = 2048L * std::max(d2c_num_cus(), 1);
    int groups = 1;
    while (groups * 2 <= std::min(a.splits, 256 / LANES) && total * LANES * groups * 2 <= places) groups *= 2;
    const long per = 256 / (LANES * groups);
    hipLaunchKernelGGL((attn_join_kernel<T, LANES>), dim3((unsigned)((total + per - 1) / per)), dim3(256), 0, st, a, groups, tile_rows);
    return d2c_check_launch("attn_join_kernel");
}
template <typename T> int launch_fwd(const d2c_attention_desc &q, const Args &a, const FwdPlan &p, hipStream_t st)
{
    const int rc = p.token ? for_token<T>(q, a.rows, [&](auto lanes, auto r, auto whole) {
        hipLaunchKernelGGL((attn_token_kernel<T, decltype(lanes)::value, decltype(r)::value, decltype(whole)::value>), dim3(workgroups(p.walks)), dim3(256), 0, st, a);
        return d2c_check_launch("attn_token_kernel");
    }) : for_shape<T>(q, p.few, [&](auto width, auto wk, auto whole) {
        constexpr int DP = decltype(width)::DP, NP = decltype(width)::NP, WK = decltype(wk)::value;
        constexpr bool WHOLE = decltype(whole)::value;
        constexpr int lds = FwdShape<T, DP, WK, WHOLE>::LDS;
        if (int e = d2c_allow_lds(reinterpret_cast<const void *>(&attn_fwd_kernel<T, DP, NP, WK, WHOLE>), lds, "attn_fwd_kernel")) return e;
        hipLaunchKernelGGL((attn_fwd_kernel<T, DP, NP, WK, WHOLE>), dim3(workgroups(p.walks)), dim3(256), lds, st, a);
        return d2c_check_launch("attn_fwd_kernel");
    });
    if (rc || p.walks.shared == 0) return rc;
    if (a.D <= 32) return launch_join<T, 8>(a, p.tile_rows, st);
    if (a.D <= 64) return launch_join<T, 16>(a, p.tile_rows, st);
    return launch_join<T, 32>(a, p.tile_rows, st);
}
template <typename T> int forward(Args a, const d2c_attention_desc &q, void *ws, size_t ws_bytes, hipStream_t st)
{
    const FwdPlan p = fwd_plan<T>(q);
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 255u))) {
        d2c_set_error("workspace of %zu bytes (256-byte aligned) required, got %zu at %p", p.bytes, ws_bytes, ws);
        return D2C_ERR_WORKSPACE;
    }
    set_walks(a, p.walks);
    a.part = (float *)ws; a.part_ml = (float *)((char *)ws + p.part_bytes);
    return launch_fwd<T>(q, a, p, st);
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
    const long heads = (long)q->N * q->Hkv, rows = (long)q->Lq * (q->Hq / q->Hkv);
    // (positions and workgroups are counted in 32 bits)
    if (heads >= (1L << 24) || rows >= (1L << 30) || q->Lk >= (1 << 30) || heads * ((std::max(rows, (long)q->Lk) + 31) / 32) >= (1L << 30)) {
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
    return a;
}

int d2c_attn::resident(const void *kernel, int lds)
{
    struct Known { const void *kernel; int dev, n; };
    static std::mutex mu;
    static Known known[512];      // (fewer kernels than this on a device; what finds no place is asked for every time)
    static int count = 0;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) { (void)hipGetLastError(); return 2; }      // (no GPU: sizes are asked for all the same)
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < count; i++)
        if (known[i].kernel == kernel && known[i].dev == dev) return known[i].n;
    int n = 0;
    if (d2c_allow_lds(kernel, lds, "attention kernel") != D2C_OK || hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, lds) != hipSuccess || n < 1) {
        (void)hipGetLastError();
        n = 1;
    }
    if (count < (int)(sizeof known / sizeof *known)) known[count++] = {kernel, dev, n};
    return n;
}

extern "C" size_t d2c_attention_forward_workspace_bytes(const d2c_attention_desc *q)
{
    if (d2c_attention_check(q) != D2C_OK || q->N == 0 || q->Lq == 0) return 0;
    return q->dtype == D2C_BF16 ? fwd_plan<bf16_t>(*q).bytes : fwd_plan<float>(*q).bytes;
}

extern "C" int d2c_attention_forward(const d2c_attention_desc *q, const void *query, const void *key, const void *value,
                                     const int32_t *key_lengths, const uint8_t *key_mask, void *out, void *out_low,
                                     float *lse, void *ws, size_t ws_bytes, void *stream)
{
    if (int rc = d2c_attention_check(q)) return rc;
    if (q->N == 0 || q->Lq == 0) return D2C_OK;
    if (!query || !out || (q->Lk > 0 && (!key || !value))) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    Args a = make_args(*q);
    a.q = query; a.k = key; a.v = value; a.lengths = key_lengths; a.mask = key_mask; a.out = out; a.lse = lse;
    a.out_low = q->dtype == D2C_BF16 ? out_low : nullptr;
    return q->dtype == D2C_BF16 ? forward<bf16_t>(a, *q, ws, ws_bytes, (hipStream_t)stream) : forward<float>(a, *q, ws, ws_bytes, (hipStream_t)stream);
}
