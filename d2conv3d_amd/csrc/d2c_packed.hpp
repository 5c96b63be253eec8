// Attention inside sequences that lie behind each other: what the forward and the backward kernels share.  Formulas and operand
// orders: d2c_attention.hpp.
//
// Where a sequence begins is known on the GPU only.  Tiles never span sequences; region i (0: what lies before the first sequence, 1 .. S: the sequences, S + 1: what
// lies behind the last) begins with tile  B_i = floor(first row / rows of a tile) + i  of one line: it has at most B_{i+1} - B_i tiles, so that a workgroup
// finds its own by the starts alone, and the line is longer than the tiles that there are by at most one tile to a region.
#pragma once
#include "d2c_attention.hpp"

namespace d2c_packed {
using namespace d2c_attn;

struct PackedArgs {
    const void *q, *k, *v, *g, *o, *o_low;
    const int32_t *starts, *key_starts;
    void *out, *out_low, *gq, *gk, *gv;
    float *lse, *delta;                     // [Hkv][T * group]
    float *part, *part_ml;                  // [splits][tiles][Hkv][128][part_width(D)] (keys' kernel: twice), and (forward) [..][2]
    long qs[2], ks[2], vs[2], gs[2];        // strides of token, head
    int T, Tk, S, Hq, Hkv, group, D, tiles, causal;
    int splits, chunk, step;                // see Walk; step: keys (rows) of a step
    FastDiv by_group, frame;
    float scale, scale2;
};

constexpr int kRows = 128;      // of a tile: rows, or keys

D2C_DEV int bound_of(const int32_t *starts, int S, int T, int i) { return i == 0 ? 0 : i > S + 1 ? T : min(max(starts[i - 1], 0), T); }
// First token of region i, and how many tokens it has
D2C_DEV void region_of(const int32_t *starts, int S, int T, int i, int &first, int &count)
{
    first = bound_of(starts, S, T, i);
    count = max((i > S ? T : bound_of(starts, S, T, i + 1)) - first, 0);
}
// The region of tile `at` of the line, which of its tiles that is, its first token and how many it has.  `group`: rows to a token.  63 regions to a vote, three votes to 250000; the last has the
// region's bounds as well.  6480 sequences of 8 tokens, 8 heads of 64, bfloat16: 436 us (448 with the bounds asked for afterwards, 1466 with regions taken 64 after 64)
D2C_DEV void find_tile(const int32_t *starts, int S, int T, int group, int at, int &region, int &tile, int &first, int &count)
{
    const int lane = threadIdx.x & 63;
    auto begin = [&](int bound, int i) INLINE { return (int)((long)bound * group / kRows) + i; };
    region = 0;
    for (int n = S + 2;;) {      // (it is one of the n regions from `region` on, whose first is known to begin in time)
        const int step = (n + 62) / 63, i = lane * step, bound = bound_of(starts, S, T, region + i);
        const int last = __builtin_ctzll(~__ballot(i < n && begin(bound, region + i) <= at)) - 1;      // (lane 63 is behind all of them)
        region += last * step;
        if (step == 1) {
            first = __builtin_amdgcn_readlane(bound, last);
            count = max(__builtin_amdgcn_readlane(bound, last + 1) - first, 0);
            break;
        }
        n = min(step, n - last * step);
    }
    tile = at - begin(first, region);
}

// A workgroup's sequence and tile
struct PackedUnit { int q0, lq, k0, lk, rows, tile, h, at, split; };
// (neighbouring workgroups have neighbouring heads, so that a head's meet in an XCD's L2 where the heads are a multiple of 8.  BY_KEYS: tiles of keys, from the first on; else tiles
// of rows, from the last on: the longest walks of a sequence come first)
template <bool BY_KEYS> D2C_DEV PackedUnit unit_of(const PackedArgs &a, int index)
{
    PackedUnit u;
    const int rest = index / a.Hkv, line = rest % a.tiles;
    u.h = index - rest * a.Hkv;
    u.split = rest / a.tiles;
    u.at = BY_KEYS ? line : a.tiles - 1 - line;
    int region, first, count;
    find_tile(BY_KEYS ? a.key_starts : a.starts, a.S, BY_KEYS ? a.Tk : a.T, BY_KEYS ? 1 : a.group, u.at, region, u.tile, first, count);
    u.q0 = u.lq = u.k0 = u.lk = 0;
    (BY_KEYS ? u.k0 : u.q0) = first;
    (BY_KEYS ? u.lk : u.lq) = count;
    if (region >= 1 && region <= a.S) {
        int &other = BY_KEYS ? u.q0 : u.k0, &others = BY_KEYS ? u.lq : u.lk;
        if (a.starts == a.key_starts && a.T == a.Tk) { other = first; others = count; }
        else region_of(BY_KEYS ? a.starts : a.key_starts, a.S, BY_KEYS ? a.T : a.Tk, region, other, others);
    }
    u.rows = u.lq * a.group;
    return u;
}
// Keys that position `pos` of a sequence reads
D2C_DEV int limit_of(const PackedArgs &a, const PackedUnit &u, int pos)
{
    if (!a.causal) return u.lk;
    const int p = u.lk - u.lq + pos;
    return p < 0 ? 0 : min(u.lk, (fdiv(p, a.frame) + 1) * a.frame.d);
}
D2C_DEV int limit_of_row(const PackedArgs &a, const PackedUnit &u, int row) { return limit_of(a, u, fdiv(row, a.by_group)); }
// The first row that reads key `key`
D2C_DEV int first_row(const PackedArgs &a, const PackedUnit &u, int key) { return a.causal ? max(fdiv(key, a.frame) * a.frame.d - (u.lk - u.lq), 0) * a.group : 0; }

// Kernels of one term of the weights (bfloat16, see kWeightTerms) take two for tiles that have sums of 64 terms or fewer, which do not average out: a tile of rows whose first reads no more
// keys, a tile of keys whose last is read by no more rows.  So results whose sums are as short, a short sequence's and those of a long one's first and last tokens, have two whatever they are
// packed with.  Such tiles' walks are short, as limits go by token or frame: forward and backward, 8 heads of 64, 500 sequences of 100 take 364 us (350 with one term everywhere), 200 of 200 281 (273);
// the longer the sequences, the fewer such tiles.  Rows of 2 to 4 keys are off by up to 0.0068 of sum p |v| with one term, by 0.0039, the result's own rounding, with two.
D2C_DEV bool few_keys(const PackedArgs &a, const PackedUnit &u) { return limit_of_row(a, u, u.tile * kRows) <= kExactKeys; }
D2C_DEV bool few_rows(const PackedArgs &a, const PackedUnit &u) { return u.rows - first_row(a, u, min(u.tile * kRows + kRows, u.lk) - 1) <= kExactKeys; }
// f(arguments, unit, terms): two bodies of a kernel, of which a workgroup takes one.  The second reads the kernel's arguments anew and has a copy of the unit that the compiler knows nothing of: it
// would take what both bodies have in common in front of the branch, and the first was 2 to 10% slower for it (products of the second term behind a branch inside the loop made kernels take 30
// to 45 registers more, or spill up to 340).
template <int TERMS, typename F> D2C_DEV void with_terms(const PackedArgs &a, const PackedUnit &u, bool few, F f)
{
    if constexpr (TERMS == 1)
        if (few) {
            auto *args = (const __attribute__((address_space(4))) PackedArgs *)__builtin_amdgcn_kernarg_segment_ptr();
            asm volatile("" : "+s"(args));
            const PackedArgs b = *(const PackedArgs *)args;
            PackedUnit w = u;
            for (int *x : {&w.q0, &w.lq, &w.k0, &w.lk, &w.rows, &w.tile, &w.h, &w.at, &w.split}) {
                *x = __builtin_amdgcn_readfirstlane(*x);
                asm volatile("" : "+s"(*x));
            }
            return f(b, w, std::integral_constant<int, 2>{});
        }
    f(a, u, std::integral_constant<int, TERMS>{});
}

// Row `row` of a tensor [tokens][Hq][D] with strides s
template <typename T> D2C_DEV const T *row_at(const void *base, const long *s, const PackedArgs &a, const PackedUnit &u, int row)
{
    const int pos = fdiv(row, a.by_group);
    return reinterpret_cast<const T *>(base) + (long)(u.q0 + pos) * s[0] + (long)(u.h * a.group + row - pos * a.group) * s[1];
}

// The keys and values of a sequence's key head, a tile of KT keys at a time
template <typename T, typename KV, int KT, bool WHOLE> struct PackedKeyTiles {
    const T *kb, *vb;
    long ks, vs;
    unsigned koff[WHOLE ? KV::PER : 1], voff[WHOLE ? KV::PER : 1];
    D2C_DEV PackedKeyTiles(const PackedArgs &a, const PackedUnit &u)
    {
        kb = reinterpret_cast<const T *>(a.k) + (long)u.k0 * a.ks[0] + u.h * a.ks[1];
        vb = reinterpret_cast<const T *>(a.v) + (long)u.k0 * a.vs[0] + u.h * a.vs[1];
        ks = a.ks[0]; vs = a.vs[0];
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < KV::PER; i++) {
                const unsigned row = KV::row_of(i), d = KV::column_of(i, a.D);
                koff[i] = (row * (unsigned)ks + d) * (unsigned)sizeof(T);
                voff[i] = (row * (unsigned)vs + d) * (unsigned)sizeof(T);
            }
        }
    }
    // left: keys of the sequence from the tile's first on (one at least); those behind repeat the last
    D2C_DEV void request(const PackedArgs &a, KV &k, KV &v, int tile, int left) const
    {
        const T *kt = kb + (long)tile * KT * ks, *vt = vb + (long)tile * KT * vs;
        if constexpr (WHOLE) {
            unsigned ko[KV::PER], vo[KV::PER];
#pragma unroll
            for (int i = 0; i < KV::PER; i++) { ko[i] = koff[i]; vo[i] = voff[i]; }
            if (left < KT) {
#pragma unroll
                for (int i = 0; i < KV::PER; i++) {
                    const unsigned step = KV::row_of(i) < left ? 0u : (unsigned)(left - 1 - KV::row_of(i)) * (unsigned)sizeof(T);
                    ko[i] += step * (unsigned)ks;
                    vo[i] += step * (unsigned)vs;
                }
            }
            k.load_at(kt, ko);
            v.load_at(vt, vo);
        } else {
            k.load(a.D, [&](int i) INLINE { return kt + min(i, left - 1) * ks; });
            v.load(a.D, [&](int i) INLINE { return vt + min(i, left - 1) * vs; });
        }
    }
};

// Whether a thread's pieces of a tile hold an infinity or NaN
template <typename T, typename Pieces> D2C_DEV bool not_finite(const Pieces &x)
{
    bool bad = false;
#pragma unroll
    for (int i = 0; i < Pieces::PER; i++)
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; j++) {
            const uint32_t w[4] = {x.r[i].v[j].x, x.r[i].v[j].y, x.r[i].v[j].z, x.r[i].v[j].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // (float32: what rounds to an infinite bfloat16 term counts as one)
                if (sizeof(T) == 4) bad = bad || (w[e] & 0x7fffffffu) > 0x7f7f7fffu;
                else bad = bad || (w[e] & 0x7f800000u) == 0x7f800000u || (w[e] & 0x7f80u) == 0x7f80u;
            }
        }
    return bad;
}

// Infinities and NaN of 16 bytes of elements (of bfloat16 terms, which an operand in LDS is made of) as zeros
D2C_DEV uint4 finite_pairs(const uint4 &x)
{
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
        if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// ... and of a thread's pieces of a tile
template <typename T, typename Pieces> D2C_DEV void clean(Pieces &x)
{
#pragma unroll
    for (int i = 0; i < Pieces::PER; i++)
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; j++) {
            if constexpr (sizeof(T) == 2) x.r[i].v[j] = finite_pairs(x.r[i].v[j]);
            else {
                uint4 &v = x.r[i].v[j];
                for (uint32_t *w : {&v.x, &v.y, &v.z, &v.w})
                    if ((*w & 0x7fffffffu) > 0x7f7f7fffu) *w = 0;
            }
        }
}
// An operand of a product whose weights are 0 where a pair is not to be read: in a tile of which some pairs are not, its infinities and NaN are left out of the product,
// whose zeros they would turn into NaN: rows r0 .. r0 + 31 of a tile in LDS, by all 256 threads between two barriers of the workgroup's ...
template <typename Pieces> D2C_DEV void clean_rows(unsigned char *lds, int r0)
{
    constexpr int ROW = Pieces::PIECES * 16;
#pragma unroll 1
    for (int i = threadIdx.x * 16; i < 32 * ROW; i += 256 * 16)
#pragma unroll 1
        for (int t = 0; t < Pieces::P; t++) {
            uint4 *p = reinterpret_cast<uint4 *>(lds + t * Pieces::TERM + r0 * ROW + i);
            *p = finite_pairs(*p);
        }
}
// ... and added once at the end, to the sums of those that read them: what a sum has once taken in stays.  x: row(j) of D, j from first to end, read(j): whether this lane's
// column reads it.  AS_NAN: what it makes whatever its weight (a key's, or query's, own infinity: its weight is NaN, or the 0 of a score of -infinity)
template <typename T, bool AS_NAN, int ND, typename Row, typename Read> D2C_DEV void take_in(f32x16 (&acc)[ND], int D, int first, int end, Row row, Read read)
{
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll 1
    for (int j = first; j < end; j++) {
        const T *p = row(j);
        const bool yes = read(j);
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int d = i * 32 + 8 * (r / 4) + 4 * half + r % 4;
                const float y = elem_to_f32<T>(p[min(d, D - 1)]);
                const bool finite = sizeof(T) == 4 ? fabsf(y) <= 0x1.fefffep127f : fabsf(y) < INFINITY;
                if (yes && !finite) acc[i][r] += AS_NAN ? NAN : y * 2.f;
                asm volatile("" : "+v"(acc[i][r]) : : "memory");      // (one value at a time)
            }
    }
}

PackedArgs make_args(const d2c_packed_attention_desc &q, const int32_t *starts, const int32_t *key_starts);
// Whether a problem runs on the kernels that load whole pieces by offsets of 32 bits inside a tile and, bfloat16, take one term of the weights but in few tiles (with_terms): not where sequences
// have 64 keys or fewer on the average, nor the backward pass where scores are few, whose errors do not average out (see kWeightTerms)
inline bool fast_kernels(const d2c_packed_attention_desc &q, bool gradients)
{
    const long average = q.keys / std::max(q.sequences, 1);
    if (q.dtype == D2C_BF16 && (average <= kExactKeys || (gradients && q.queries * q.Hq <= kExactScores / average))) return false;
    const long size = (long)d2c_elem_size(q.dtype), limit = 1L << 31;
    auto near = [&](const int64_t *s) { return s[0] >= 0 && s[1] >= 0 && 129 * s[0] * size + (q.Hq / q.Hkv) * s[1] * size < limit; };
    return q.D % 8 == 0 && near(q.q_stride) && near(q.k_stride) && near(q.v_stride) && 130L * q.Hq * q.D * size < limit;
}
inline int tiles_of(long rows, int sequences) { return (int)(rows / kRows) + sequences + 2; }

// The steps of a unit's walk, and how many workgroups share it: as many as make pieces of `chunk` steps, `splits` at most.  Long walks beside short ones (a sequence's last
// rows beside its first, its first keys beside its last) would be what the GPU waits for in the end.
struct Walk { int first, steps, splits; };
D2C_DEV Walk walk_of(const PackedArgs &a, int first, int steps) { return {first, steps, min(max((steps + a.chunk - 1) / a.chunk, 1), a.splits)}; }
// ... of rows: keys up to the last that the last of them reads
D2C_DEV Walk row_walk(const PackedArgs &a, const PackedUnit &u)
{
    const int row0 = u.tile * kRows;
    return walk_of(a, 0, row0 < u.rows ? (limit_of_row(a, u, min(row0 + kRows, u.rows) - 1) + a.step - 1) / a.step : 0);
}
// ... of keys: rows from the first that reads the first of them
D2C_DEV Walk key_walk(const PackedArgs &a, const PackedUnit &u)
{
    const int first = first_row(a, u, u.tile * kRows) / a.step;
    return walk_of(a, first, max((u.rows + a.step - 1) / a.step - first, 0));
}
// On the host, where only the average length is known: the longest walk is taken to be twice that of a sequence of the average length, or that of the only sequence.  Pieces cost a second
// launch and their sums' way through memory, so walks are cut where one is longer than what every place gets anyway, into pieces of a third of that: one sequence of 25920, forward and backward,
// 3.37 ms (when this was chosen 3.44; 4.99 whole, 3.95 in pieces of three quarters, 3.67 of a fifth); six of up to 12960 2.95 (then 2.98; 3.07 to 3.16 in pieces).  One long sequence beside many short
// ones, whose average says nothing of it, is not cut.
struct Split { int splits, chunk; };
inline Split split_walks(const d2c_packed_attention_desc &q, long units, long places, long along, long step, double unit_bytes)
{
    const long sequences = std::max(q.sequences, 1), average = along / sequences / step + 1, longest = sequences == 1 ? average : 2 * average;
    const double each = (double)units * (double)average * (q.causal ? 0.5 : 1.0) / (double)places;      // steps that every place gets
    if ((double)longest <= 1.25 * each) return {1, 1 << 30};
    // (of 4 steps at least where all of them have a place at once, else of 8: four sequences of up to 350, float32, 14.3 us in pieces of 4, 18.7 of 8; three of up to 1417, forward and backward, 134 in
    // pieces of 4, 121 of 6 or 8, 145 of 12)
    const long chunk = std::max((long)(each * 0.3), units * (longest / 4 + 1) * (q.causal ? 1 : 2) <= 2 * places ? 4L : 8L);
    long s = std::min((longest + chunk - 1) / chunk, 16L);
    while (s > 1 && (double)s * (double)units * unit_bytes > part_limit(q)) s--;
    return {(int)s, s > 1 ? (int)chunk : 1 << 30};
}

}  // namespace d2c_packed

int d2c_packed_attention_check(const d2c_packed_attention_desc *q);
