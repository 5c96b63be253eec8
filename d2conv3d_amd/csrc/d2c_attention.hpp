// Building blocks of the attention kernels: operand fragments, tiles in LDS, the mapping of rows.
//
//   s[i][j] = scale * sum_d q[i][d] k[j][d]   over the keys j that are there
//   p = exp(s - max_j s) / sum_j exp(s - max_j s),   o[i] = sum_j p[i][j] v[j]           (a row without a key: o = 0)
//   backward, with L = log sum_j exp s kept from the forward pass and delta = sum_d do[i][d] o[i][d]:
//     p = exp(s - L),  dv = p^T do,  dp = do v^T,  ds = p (dp - delta),  dq = scale ds k,  dk = scale ds^T q
//
// Everything runs on v_mfma_f32_32x32x16_bf16.  The scores are made with the reader's index along the lanes (one column of the
// accumulator to a lane): row maxima and sums then stay in a lane but for one exchange between its halves, and the
// accumulator's registers are the next product's operand as they are -- in the order of the reduction that the accumulator has,
// 4 of 8 keys to a half of the wavefront, in which the other operand is read, too (transposing LDS reads, four at a time).
//
// float32 operands travel as three bfloat16 terms, which represent a float exactly, and a product as the six partial products that
// count (what is left out is below 2^-24 of it): 6/16 of the float instruction's time.
//
// The rows of a group of query heads that share a key head are one axis: row = position * group + head in group.
#pragma once
#include <algorithm>
#include <type_traits>
#include "d2c_common.hpp"
#include "d2c_mma.hpp"

namespace d2c_attn {

struct Args {
    const void *q, *k, *v, *g, *o;      // g: gradient of the output o
    const void *o_low;                  // what rounding took off o (bfloat16, or NULL)
    const int32_t *lengths;             // [N] or NULL
    const uint8_t *mask;                // [N][Lk], 0: not to be read; or NULL
    void *out, *gq, *gk, *gv;           // [N][Lq][Hq][D], [N][Lk][Hkv][D]
    void *out_low;                      // NULL, or where the forward pass leaves o_low
    float *lse, *delta;                 // [N * Hkv][rows]: log2 of the sum of a row (+infinity: no key), and sum_d do o
    float *part, *part_ml;              // partial results of the walks that are shared: [splits][shared][rows of a tile][D] and (forward) [..][2]
    long qs[3], ks[3], vs[3], gs[3];    // strides of sample, position, head
    int N, Lq, Lk, Hq, Hkv, group, D, rows;
    int whole, shared, splits;          // see Walks
    float scale, scale2;                // scale2 = scale * log2(e)
};

template <typename T> constexpr int kTerms = sizeof(T) == 2 ? 1 : 3;
// Terms of the weights p and of ds, which are rounded to the matrix instruction's operands: bfloat16 problems take one, whose errors (2^-9 of each; the row's sum is
// that of the weights before) are as large as the rounding of the result and average out over many keys: 2.4e-3 of a result in all, 1.7e-3 of them by its own
// rounding.  A second term everywhere would take 1.34 to 1.45 times as long (1620 rows on 64800 keys of 8 heads of 128, 470, 628 us; 12960 on 25920 of 64,
// forward and backward, 3260, 4717).  Where a call has 64 keys or fewer, errors do not average out (two keys: weights just above 1/2, where the spacing is
// widest), nor in the gradients of a small problem: these have the second term, at 1.11 to 1.16 times the backward kernels' time where the line is (512 rows on
// 1024 keys of 8 heads of 64, 38.1, 42.9 us; of 128, 54.6, 63.0; whole passes are the host's 55 to 85 us either way).  Calls count, not samples: two keys that a mask leaves
// of 1000 have weights of one term in a large call.  (Heads of an odd size, and rows that lie further apart than 32-bit offsets reach, run on the same kernels and have it, too.)
template <typename T, bool FAST> constexpr int kWeightTerms = sizeof(T) == 4 ? 3 : FAST ? 1 : 2;
constexpr int kExactKeys = 64;
constexpr long kExactScores = 1L << 22;

// 8 reduction elements of a matrix operand's row
template <int P> struct Frag { uint4 t[P]; };

D2C_DEV f32x16 mma1(f32x16 acc, const uint4 &a, const uint4 &b)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc, 0, 0, 0);
}
template <int P, int PB> D2C_DEV void mma(f32x16 &acc, const Frag<P> &a, const Frag<PB> &b)
{
    static_assert(P == 1 || PB == 3, "");
    if constexpr (P == 1 && PB == 2) acc = mma1(acc, a.t[0], b.t[1]);
    if constexpr (P == 3) {
        acc = mma1(acc, a.t[2], b.t[0]);
        acc = mma1(acc, a.t[0], b.t[2]);
        acc = mma1(acc, a.t[1], b.t[1]);
        acc = mma1(acc, a.t[1], b.t[0]);
        acc = mma1(acc, a.t[0], b.t[1]);
    }
    acc = mma1(acc, a.t[0], b.t[0]);
}
// Two floats -> their three terms, each a packed pair.  INFINITIES (operands that come from memory): one, or a value that rounds to one, is the last term alone.  It
// meets the other operand's first term only, which is 0 where the value is and has its sign, and so makes the infinity that the product is; against lower
// terms, which are 0 or of either sign, it would make no number.
template <bool INFINITIES> D2C_DEV void split_pair(float x, float y, uint32_t &hi, uint32_t &mid, uint32_t &lo)
{
    const bool ix = INFINITIES && fabsf(x) > 0x1.fefffep127f, iy = INFINITIES && fabsf(y) > 0x1.fefffep127f;
    const float x0 = ix ? 0.f : x, y0 = iy ? 0.f : y;
    hi = pack_bf16x2(x0, y0);
    const float x1 = x0 - __uint_as_float(hi << 16), y1 = y0 - __uint_as_float(hi & 0xffff0000u);
    mid = pack_bf16x2(x1, y1);
    const float x2 = x1 - __uint_as_float(mid << 16), y2 = y1 - __uint_as_float(mid & 0xffff0000u);
    lo = pack_bf16x2(ix ? x : x2, iy ? y : y2);
}
// ... their two terms
D2C_DEV void split_pair(float x, float y, uint32_t &hi, uint32_t &lo)
{
    hi = pack_bf16x2(x, y);
    lo = pack_bf16x2(bf16_residual(x, hi << 16), bf16_residual(y, hi & 0xffff0000u));
}
// ... which agree in sign and neither of which is 0 where the value is not (down to 2^-86: what a second term of 0 would be is 2^-40 of the value).  The other
// operand is one term: an infinite one makes the infinity that the product is of both.
D2C_DEV void split_pair_agreeing(float x, float y, uint32_t &hi, uint32_t &lo)
{
    auto behind = [](float v) INLINE { return fmaf(v, 0x1p-40f, v - __uint_as_float(__float_as_uint(v) & 0xffff0000u)); };
    hi = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
    lo = pack_bf16x2(behind(x), behind(y));
}
// Operands that the kernels make (WEIGHTS: those, whose other operand may be infinite; never infinite themselves) or that come from memory
enum Operand { MADE, WEIGHTS, READ };
template <int P, Operand KIND> D2C_DEV Frag<P> make_frag(const float *v)
{
    Frag<P> f;
    if constexpr (P == 2 && KIND == WEIGHTS) {
        uint32_t h[4], m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_pair_agreeing(v[2 * i], v[2 * i + 1], h[i], m[i]);
        f.t[0] = make_uint4(h[0], h[1], h[2], h[3]);
        f.t[1] = make_uint4(m[0], m[1], m[2], m[3]);
    } else if constexpr (P == 1) {
        f.t[0] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else if constexpr (P == 2) {
        uint32_t h[4], m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_pair(v[2 * i], v[2 * i + 1], h[i], m[i]);
        f.t[0] = make_uint4(h[0], h[1], h[2], h[3]);
        f.t[1] = make_uint4(m[0], m[1], m[2], m[3]);
    } else {
        uint32_t h[4], m[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_pair<KIND == READ>(v[2 * i], v[2 * i + 1], h[i], m[i], l[i]);
        f.t[0] = make_uint4(h[0], h[1], h[2], h[3]);
        f.t[1] = make_uint4(m[0], m[1], m[2], m[3]);
        f.t[2] = make_uint4(l[0], l[1], l[2], l[3]);
    }
    return f;
}

// 8 elements as they lie in memory.  WHOLE: all of them there; else `left` of them (zeros behind; none: p is not read)
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };
template <bool WHOLE, typename T> D2C_DEV Raw8<T> load8(const T *p, int left)
{
    constexpr int VEC = 16 / (int)sizeof(T);
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) {
        if constexpr (WHOLE) {
            const AnyVec<T> v = load_any(p + i * VEC);
            r.v[i] = make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            r.v[i] = make_uint4(0, 0, 0, 0);
            if (left > i * VEC) r.v[i] = load_run<T>(p + i * VEC, left - i * VEC);
        }
    }
    return r;
}
// ... of a row of D elements, from element d on, zeros behind the row (WHOLE: D is a multiple of 8)
template <bool WHOLE, typename T> D2C_DEV Raw8<T> load8_of(const T *row, int d, int D, bool live)
{
    if constexpr (WHOLE) {
        Raw8<T> r = load8<true, T>(row + min(d, D - 8), 8);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            if (d >= D || !live) r.v[i] = make_uint4(0, 0, 0, 0);
        return r;
    } else return load8<false, T>(row + d, live ? D - d : 0);
}
template <typename T> D2C_DEV Frag<kTerms<T>> terms_of(const Raw8<T> &r)
{
    if constexpr (sizeof(T) == 2) return Frag<1>{{r.v[0]}};
    else {
        float f[8];
        *reinterpret_cast<uint4 *>(f) = r.v[0];
        *reinterpret_cast<uint4 *>(f + 4) = r.v[1];
        return make_frag<3, READ>(f);
    }
}
template <typename T> D2C_DEV void floats_of(const Raw8<T> &r, float *f)
{
    if constexpr (sizeof(T) == 2) {
        const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
        for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else {
        *reinterpret_cast<uint4 *>(f) = r.v[0];
        *reinterpret_cast<uint4 *>(f + 4) = r.v[1];
    }
}

// A tile of ROWS rows of DP bfloat16 values (per term) in LDS, in pieces of 16 bytes.  A row's pieces change places so that neither 8
// rows' pieces of one column (operand reads) nor 4 rows' 64 bytes (transposing reads) meet in a bank.
template <int DP> D2C_DEV int piece_swizzle(int row)
{
    if constexpr (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (DP == 64) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
}
template <int DP> D2C_DEV int piece_at(int row, int piece) { return row * (DP * 2) + ((piece ^ piece_swizzle<DP>(row)) << 4); }

typedef short v4s_t __attribute__((ext_vector_type(4)));

// WHOLE (heads are whole pieces, rows near enough for offsets of 32 bits): loads without branches.  Pieces behind a row's end then repeat its last one and make
// columns that are not stored.  Else elements behind the end are zeros.
template <typename T, int DP, int ROWS, int THREADS, bool WHOLE> struct Tile {
    static constexpr int P = kTerms<T>, PIECES = DP / 8, PER = (ROWS * PIECES + THREADS - 1) / THREADS;
    static constexpr int TERM = ROWS * DP * 2, BYTES = P * TERM;
    Raw8<T> r[PER];
    // this thread's piece i: its row and first column
    static D2C_DEV int place(int i) { return min(i * THREADS + (int)threadIdx.x, ROWS * PIECES - 1); }
    static D2C_DEV int row_of(int i) { return place(i) / PIECES; }
    static D2C_DEV int column_of(int i, int D) { return WHOLE ? min(place(i) % PIECES * 8, D - 8) : place(i) % PIECES * 8; }
    // row(i): the address of row i, which is there to be read whatever i
    template <typename Row> D2C_DEV void load(int D, Row row)
    {
        static_assert(!WHOLE, "");
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int d = column_of(i, D);
            r[i] = load8<false, T>(row(row_of(i)) + d, D - d);
        }
    }
    // WHOLE: by offsets in bytes from one address
    D2C_DEV void load_at(const T *base, const unsigned (&off)[PER])
    {
#pragma unroll
        for (int i = 0; i < PER; i++) r[i] = load8<true, T>(reinterpret_cast<const T *>(reinterpret_cast<const char *>(base) + off[i]), 8);
    }
    // zeros in the rows that drop(row) says
    template <typename Drop> D2C_DEV void zero_rows(Drop drop)
    {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const bool gone = drop(row_of(i));
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; j++)
                if (gone) r[i].v[j] = make_uint4(0, 0, 0, 0);
        }
    }
    // END: the piece at column D, which a product's last step takes in, as zeros (those of the other operand do not undo an infinity that is repeated)
    template <bool END> D2C_DEV void store(unsigned char *lds, int D) const
    {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int at = i * THREADS + threadIdx.x;
            if (ROWS * PIECES % THREADS != 0 && at >= ROWS * PIECES) continue;
            Raw8<T> x = r[i];
            if constexpr (END) {
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) / 2; j++)
                    if (at % PIECES * 8 == D) x.v[j] = make_uint4(0, 0, 0, 0);
            }
            const Frag<P> f = terms_of<T>(x);
#pragma unroll
            for (int t = 0; t < P; t++)
                *reinterpret_cast<uint4 *>(lds + t * TERM + piece_at<DP>(at / PIECES, at % PIECES)) = f.t[t];
        }
    }
    // columns 16 ks + 8 half .. of row `row`
    static D2C_DEV Frag<P> rows(const unsigned char *lds, int row, int ks, int half)
    {
        Frag<P> f;
#pragma unroll
        for (int t = 0; t < P; t++) f.t[t] = *reinterpret_cast<const uint4 *>(lds + t * TERM + piece_at<DP>(row, ks * 2 + half));
        return f;
    }
    // column c0 + lane % 32 of the rows r0 + {0..3, 8..11} (first half of the wavefront) and r0 + {4..7, 12..15}: the order in which an
    // accumulator's registers 8 i .. 8 i + 7 hold them.  (Within 16 lanes, lane l element j comes from lane 4j + l/4, element l%4.)
    static D2C_DEV Frag<P> columns(const unsigned char *lds, int r0, int c0, int lane)
    {
        const int row = r0 + (lane >> 5) * 4 + ((lane & 15) >> 2), col = c0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        Frag<P> f;
#pragma unroll
        for (int t = 0; t < P; t++) {
            const unsigned char *p = lds + t * TERM + (col & 7) * 2;
            const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_t *)(p + piece_at<DP>(row, col >> 3))));
            const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_t *)(p + piece_at<DP>(row + 8, col >> 3))));
            f.t[t] = make_uint4(a.x, a.y, b.x, b.y);
        }
        return f;
    }
};

// Widths that kernels are made for: channels of a tile, a multiple of 32 (the products' columns), and pieces of 8 that heads have (the widest's where they are no
// whole pieces).  The products over channels take NK steps of 16, the last of which may have one piece alone (END).
// A last step that heads do not reach is left out (8000 on 8000 positions of 8 heads, bfloat16, forward and backward, us: 40 channels 203 + 586, 191 + 557; 104
// channels 274 + 981, 266 + 856; 1417 on 3001 of 6 heads of 40, float32: the three kernels 210, 181).
template <int DP_, int NP_> struct Width { static constexpr int DP = DP_, NP = NP_; };
template <int NP> constexpr int kSteps = (NP + 1) / 2;
// Whether a problem runs on the kernels that load whole pieces by offsets of 32 bits: of a tile of 128 keys at most, of all rows (and, bfloat16, take one term of
// the weights)
inline bool fast_kernels(const d2c_attention_desc &q, bool gradients)
{
    if (q.dtype == D2C_BF16 && (q.Lk <= kExactKeys || (gradients && (long)q.N * q.Hq * q.Lq <= kExactScores / q.Lk))) return false;
    const long size = (long)d2c_elem_size(q.dtype), limit = 1L << 31;
    auto keys_near = [&](long stride) { return stride >= 0 && 128 * stride * size < limit; };
    auto rows_near = [&](const int64_t *s) { return s[1] >= 0 && s[2] >= 0 && (q.Lq * s[1] + q.Hq / q.Hkv * s[2] + q.D) * size < limit; };
    const int64_t g[3] = {0, (int64_t)q.Hq * q.D, q.D};
    return q.D % 8 == 0 && keys_near(q.k_stride[1]) && keys_near(q.v_stride[1]) && rows_near(q.q_stride) && rows_near(g);
}
template <typename T, bool GRADIENTS, typename F> auto for_width(const d2c_attention_desc &q, F f)      // f(Width, fast_kernels)
{
    const int pieces = (q.D + 7) / 8;
    auto pick = [&](auto width) {      // (of the four widths with as many channels)
        constexpr int DP = decltype(width)::DP, NP = DP / 8;
        if (!fast_kernels(q, GRADIENTS)) return f(Width<DP, NP>{}, std::false_type{});
        if (pieces == NP - 3) return f(Width<DP, NP - 3>{}, std::true_type{});
        if (pieces == NP - 2) return f(Width<DP, NP - 2>{}, std::true_type{});
        if (pieces == NP - 1) return f(Width<DP, NP - 1>{}, std::true_type{});
        return f(Width<DP, NP>{}, std::true_type{});
    };
    if (pieces <= 4) return pick(Width<32, 4>{});
    if (pieces <= 8) return pick(Width<64, 8>{});
    if (pieces <= 12) return pick(Width<96, 12>{});
    return pick(Width<128, 16>{});
}

// Floats to a row of partial sums: whole pieces of 16 bytes (what is behind a row's end is read and dropped)
inline __host__ __device__ int part_width(int D) { return (D + 3) & ~3; }

// What the workgroups do: units, each the walk of one tile of rows (or keys) of one key head along the other axis.  As many as
// fill the GPU's places without a remainder are walked by a workgroup each (`whole`); `splits` workgroups share each of the `shared` others, so that the
// last round is as short as it is empty, and their sums are joined.
// Consecutive units are of consecutive heads, so that a head's workgroups meet in an XCD's L2 where the heads are a multiple of 8.
struct Walks { int whole, shared, splits; };
struct Head { int n, h; long nh; };
struct Unit { Head head; int tile, split, splits, part; };      // part: which of the shared ones, for split 0
D2C_DEV Unit unit_of(const Args &a)
{
    int unit = (int)blockIdx.x, split = 0, splits = 1, part = 0;
    if (unit >= a.whole) {
        const int i = unit - a.whole;
        split = i / a.shared;
        part = i - split * a.shared;
        unit = a.whole + part;
        splits = a.splits;
    }
    const int heads = a.N * a.Hkv, tile = unit / heads, nh = unit - tile * heads, n = nh / a.Hkv;
    return {{n, nh - n * a.Hkv, nh}, tile, split, splits, part};
}
// ... of `steps` steps of `step_us` each at the places' full number, `bytes` of partial sums to a unit and split, `limit` bytes in all.  Times of the model: 4 us
// for the launch that joins, its traffic (written and read) at 4 TB/s.  (Without a limit 20000 rows of one head of 128 reading 2^24 keys would ask for 770
// MB, to fill a last round's idle places.  Of 10000 calls of up to 12960 rows and 64800 keys, drawn at random, two would ask for more than 256 MB.)
inline Walks plan_walks(long units, long steps, long places, double step_us, double bytes, double limit)
{
    Walks w{(int)(units / places * places), 0, 1};
    w.shared = (int)(units - w.whole);
    if (w.shared == 0) return w;
    double best = 0.0;
    for (long s = 1; s <= std::max(std::min(steps, 256L), 1L); s++) {
        if (s > 1 && (double)(w.shared * s) * bytes > limit) break;
        const double t = (double)((w.shared * s + places - 1) / places) * (double)((steps + s - 1) / s) * step_us +
                         (s > 1 ? 4.0 + 2.0 * (double)(w.shared * s) * bytes / 4e6 : 0.0);
        if (s == 1 || t < best) { best = t; w.splits = (int)s; }
    }
    if (w.splits == 1) { w.whole += w.shared; w.shared = 0; }
    return w;
}
inline double part_limit(const d2c_attention_desc &q) { return q.part_limit == 0 ? (double)D2C_ATTENTION_PART_BYTES : (double)q.part_limit; }
inline unsigned workgroups(const Walks &w) { return (unsigned)(w.whole + w.shared * w.splits); }
// Workgroups of a kernel that a compute unit holds
int resident(const void *kernel, int lds);

D2C_DEV int keys_of(const Args &a, int n) { return a.lengths ? min(max(a.lengths[n], 0), a.Lk) : a.Lk; }

// A sample of up to 64 keys (by its length) of which one is to be read: its weight is 1 whatever its score, and the score's gradients are 0, not what two sums of
// the same terms in different orders leave (as they do where a mask leaves one of more keys: 2^-24 of the terms for each channel).
D2C_DEV bool one_key(const Args &a, int n, int keys)
{
    if (keys > kExactKeys) return false;
    const int key = threadIdx.x & 63;
    return __popcll(__ballot(key < keys && (!a.mask || a.mask[(long)n * a.Lk + key]))) == 1;
}

// Row `row` of a tensor [N][Lq][Hq][D] with strides s
template <typename T> D2C_DEV const T *row_at(const void *base, const long *s, const Args &a, const Head &hd, int row)
{
    const int pos = row / a.group, g = row - pos * a.group;
    return reinterpret_cast<const T *>(base) + hd.n * s[0] + pos * s[1] + (long)(hd.h * a.group + g) * s[2];
}

// Four consecutive values of a row that ends at `left`
template <typename T> D2C_DEV void store4(T *p, const float *v, int left)
{
    typedef uint32_t u32x2_by2 __attribute__((ext_vector_type(2), aligned(2)));
    typedef float f32x4_by4 __attribute__((ext_vector_type(4), aligned(4)));
    if (left >= 4) {
        if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2_by2 *>(p) = u32x2_by2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        else *reinterpret_cast<f32x4_by4 *>(p) = f32x4_by4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) p[i] = f32_to_elem<T>(v[i]);
    }
}

// ... what storing them as T takes off
template <typename T> D2C_DEV void store4_low(T *p, const float *v, int left)
{
    float low[4];
#pragma unroll
    for (int i = 0; i < 4; i++) low[i] = v[i] - elem_to_f32<T>(f32_to_elem<T>(v[i]));
    store4<T>(p, low, left);
}

// Both halves of the wavefront: the larger value, the sum
D2C_DEV void other_half(float v, float &x, float &y)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    x = __uint_as_float(r[0]); y = __uint_as_float(r[1]);
}
D2C_DEV float half_max(float v) { float x, y; other_half(v, x, y); return fmaxf(x, y); }
D2C_DEV float half_sum(float v) { float x, y; other_half(v, x, y); return x + y; }

// The rows of a tile of keys to request: a key that is not to be read is replaced by one of the tile's that is (any_key, of `words`), so that
// what it holds is nowhere read: its score is put to -infinity, and its weight 0 meets zeros that are put in the place of that other key's value (which
// may be infinite).
template <int WORDS> D2C_DEV bool has_key(const uint64_t (&words)[WORDS], int i)
{
    const uint64_t w = WORDS == 1 ? words[0] : words[i >> 6];
    return (w >> (i & 63)) & 1;
}
template <int KT, int WORDS> D2C_DEV bool all_keys(const uint64_t (&words)[WORDS])
{
    bool all = true;
#pragma unroll
    for (int j = 0; j < WORDS; j++) all = all && words[j] == (KT < 64 ? (1ull << (KT & 63)) - 1 : ~0ull);
    return all;
}
template <int WORDS> D2C_DEV int any_key(const uint64_t (&words)[WORDS])
{
#pragma unroll
    for (int j = 0; j < WORDS; j++)
        if (words[j]) return j * 64 + __builtin_ctzll(words[j]);
    return -1;
}

Args make_args(const d2c_attention_desc &q);

// The keys and values of one key head, a tile of KT keys at a time
template <typename T, typename KV, int KT, int WORDS, bool WHOLE> struct KeyTiles {
    const T *kb, *vb;
    long ks, vs;
    unsigned koff[WHOLE ? KV::PER : 1], voff[WHOLE ? KV::PER : 1];
    D2C_DEV KeyTiles(const Args &a, const Head &hd)
    {
        kb = reinterpret_cast<const T *>(a.k) + hd.n * a.ks[0] + hd.h * a.ks[2];
        vb = reinterpret_cast<const T *>(a.v) + hd.n * a.vs[0] + hd.h * a.vs[2];
        ks = a.ks[1]; vs = a.vs[1];
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < KV::PER; i++) {
                const unsigned row = KV::row_of(i), d = KV::column_of(i, a.D);
                koff[i] = (row * (unsigned)ks + d) * (unsigned)sizeof(T);
                voff[i] = (row * (unsigned)vs + d) * (unsigned)sizeof(T);
            }
        }
    }
    // `words`: the tile's keys that are to be read (none: nothing is requested)
    D2C_DEV void request(const Args &a, KV &k, KV &v, int tile, const uint64_t (&words)[WORDS]) const
    {
        const int any = any_key(words);
        if (any < 0) return;
        const T *kt = kb + (long)tile * KT * ks, *vt = vb + (long)tile * KT * vs;
        if constexpr (WHOLE) {
            unsigned ko[KV::PER], vo[KV::PER];
            const bool all = all_keys<KT>(words);
#pragma unroll
            for (int i = 0; i < KV::PER; i++) { ko[i] = koff[i]; vo[i] = voff[i]; }
            if (!all) {
#pragma unroll
                for (int i = 0; i < KV::PER; i++) {
                    const unsigned step = has_key(words, KV::row_of(i)) ? 0u : (unsigned)(any - KV::row_of(i)) * (unsigned)sizeof(T);
                    ko[i] += step * (unsigned)ks;
                    vo[i] += step * (unsigned)vs;
                }
            }
            k.load_at(kt, ko);
            v.load_at(vt, vo);
        } else {
            k.load(a.D, [&](int i) INLINE { return kt + (has_key(words, i) ? i : any) * ks; });
            v.load(a.D, [&](int i) INLINE { return vt + (has_key(words, i) ? i : any) * vs; });
        }
    }
};
inline void set_walks(Args &a, const Walks &w) { a.whole = w.whole; a.shared = w.shared; a.splits = w.splits; }

}  // namespace d2c_attn

int d2c_attention_check(const d2c_attention_desc *q);
