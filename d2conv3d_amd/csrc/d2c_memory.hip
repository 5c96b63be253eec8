// A memory of keys and values in pages: tokens appended, read by one new token of each stream, evicted by accumulated weight.
//
//   attention  s_j = scale <q, k_j>,  p_j = exp(s_j - max s) / sum exp(s - max s),  o = sum_j p_j v_j,  usage_j += sum over rows of p_j
//   eviction   a slot stays if its token is one of the newest, or if its usage is among the largest of the others
#include <type_traits>
#include "d2c_attention.hpp"

using namespace d2c_attn;

namespace {

struct MemArgs {
    const void *q;
    void *key, *value, *out;
    const int32_t *table, *lengths;
    float *usage;                 // or NULL
    float *part, *part_ml;        // [units + places][R][part_width(D)], and (maximum, sum) of each row
    int32_t *covered;             // [units][2]: the first and the last workgroup that has a piece of the unit
    int32_t *begins;              // [places][4]: unit and step that a workgroup begins with, its steps
    float *scores;                // [units][slots][score_rows], or [units][score_rows][slots], of base 2
    long qs[2], ks[3], vs[3], table_stride, slots_padded;
    FastDiv page;
    int N, heads, group, D, pages, slots, row_groups, units, places, least, score_rows;
    float scale2;
};

D2C_DEV int slots_of(const MemArgs &a, int n) { return min(max(a.lengths[n], 0), a.slots); }
// Steps of a stream's walk: one at least, so that a stream without slots has a unit that writes its zeros
template <int STEP> D2C_DEV int steps_of(const MemArgs &a, int n) { return max(1, (slots_of(a, n) + STEP - 1) / STEP); }

// Sum over the lanes up to this one, without LDS
template <int CTRL, int ROWS> D2C_DEV int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
D2C_DEV int wave_scan(int v)
{
    v = dpp_add<0x111, 0xf>(v);      // inside rows of sixteen lanes: from 1, 2, 4, 8 lanes before
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);      // the second and fourth row: the last lane of the row before
    v = dpp_add<0x143, 0xc>(v);      // the upper half: the last lane of the lower
    return v;
}
// ... of a wavefront's sums, those before `wave`: all requested at once
template <int WAVES> D2C_DEV int before_wave(const int *sums, int wave)
{
    int x = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) x += w < wave ? sums[w] : 0;
    return x;
}

// Where this workgroup begins.  The steps of all units (stream, key head, rows of up to eight; in this order) are one line, of which every workgroup takes as
// many as the others: streams of any lengths load all compute units alike, and no length is known on the host.  False: nothing left for this one.
template <int STEP> D2C_DEV bool find_begin(const MemArgs &a, int &unit, int &t, int &budget)
{
    __shared__ int s_wave[4], s_found[2];
    const int tid = threadIdx.x, wave = tid >> 6, per_stream = a.heads * a.row_groups;
    int c = 0;
    for (int n = tid; n < a.N; n += 256) c += steps_of<STEP>(a, n);
    int scan = wave_scan(c);
    if ((tid & 63) == 63) s_wave[wave] = scan;
    __syncthreads();
    const long total = (long)(s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3]) * per_stream;
    budget = max((int)((total + a.places - 1) / a.places), a.least);
    const long start = (long)blockIdx.x * budget;
    if (start >= total) return false;
    long base = 0;
    for (int n0 = 0; n0 < a.N; n0 += 256) {
        const int n = n0 + tid;
        if (a.N > 256) {
            c = n < a.N ? steps_of<STEP>(a, n) : 0;
            scan = wave_scan(c);
            __syncthreads();
            if ((tid & 63) == 63) s_wave[wave] = scan;
            __syncthreads();
        }
        const long before = base + scan - c + before_wave<4>(s_wave, wave);
        if (n < a.N && before * per_stream <= start && start < (before + c) * per_stream) { s_found[0] = n; s_found[1] = (int)before; }
        base += s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
    }
    __syncthreads();
    const int n = s_found[0], steps = steps_of<STEP>(a, n), off = (int)(start - (long)s_found[1] * per_stream);
    unit = n * per_stream + off / steps;
    t = off % steps;
    return true;
}

// The weights of a key head's slots from s0 to s1, added up over all its rows, R to a unit.  s_ml: maximum and 1 / sum of the rows.  Scores lie slot by slot, a unit's rows
// together, or (PLANES) row by row
template <int R, bool PLANES> D2C_DEV void add_usage(const MemArgs &a, int unit, int n, int h, int s0, int s1, const float2 *s_ml)
{
    for (int s = s0 + (int)threadIdx.x; s < s1; s += 256) {
        const int p = fdiv(s, a.page), id = a.table[n * a.table_stride + p];
        if ((unsigned)id >= (unsigned)a.pages) continue;
        float *to = a.usage + ((long)id * a.heads + h) * a.page.d + (s - p * a.page.d);
        const float old = *to;
        float x = 0.f;
        for (int g = 0; g < a.row_groups; g++) {
            const float *from = a.scores + (long)(unit + g) * a.slots_padded * a.score_rows;
            if constexpr (PLANES) {
                const int rows = min(R, a.group - g * R);
#pragma unroll 4
                for (int r = 0; r < rows; r++) x += __builtin_amdgcn_exp2f(from[r * a.slots_padded + s] - s_ml[g * R + r].x) * s_ml[g * R + r].y;
            } else {
                float score[R];
                from += (long)s * R;
                if constexpr (R % 4 == 0) {
#pragma unroll
                    for (int r = 0; r < R; r += 4) *reinterpret_cast<float4 *>(score + r) = *reinterpret_cast<const float4 *>(from + r);
                } else {
#pragma unroll
                    for (int r = 0; r < R; r++) score[r] = from[r];
                }
#pragma unroll
                for (int r = 0; r < R; r++)
                    if (g * R + r < a.group) x += __builtin_amdgcn_exp2f(score[r] - s_ml[g * R + r].x) * s_ml[g * R + r].y;
            }
        }
        *to = old + x;
    }
}
// (a row whose sum is 0 has no slot, or none whose score is above -infinity: no weights)
D2C_DEV float2 usage_ml(float top, float sum) { return make_float2(top == -INFINITY ? 0.f : top, sum == 0.f ? 0.f : 1.f / sum); }

// One new token of each stream.  As attn_token_kernel, by lanes and without matrix instructions: LANES lanes hold a slot's key and value, 16 bytes each, a wavefront
// 64 / LANES slots; every group of lanes keeps its own maximum, sum and output of each of the R rows until the end of the unit's piece.  The page of a slot is
// asked for two steps ahead, its key and value one.  ONE: a workgroup to a unit (short memories), which needs no second launch.
// Bound: memory.  Measured, bfloat16, four rows: two streams of 129600 slots, 2 heads of 128, pages of 64 in any order, 54.8 us (265 MB, 4.8 TB/s; a copy 5.1) and the join 5.6; 32 streams of up
// to 12960, 4 heads of 64, with scores written for the weights, 55 us (222 MB).  Three workgroups to a compute unit instead of two are 3 us longer on the first and no shorter on the second.
template <typename T, int LANES, int R, bool WHOLE, bool ONE> __global__ void __launch_bounds__(256) mem_attn_kernel(MemArgs a)
{
    using Shape = TokenShape<T, LANES, R>;
    constexpr int VEC = Shape::VEC, DP = Shape::DP, LOADS = Shape::LOADS, KEYS = Shape::KEYS, STEP = Shape::STEP;
    __shared__ __align__(16) float s_o[4][R][DP];
    __shared__ float2 s_ml[4][R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d0 = lane % LANES * VEC;
    // (ONE: with weights to add up, all groups of a key head's rows one after the other)
    __shared__ float2 s_row[ONE ? 256 : 1];
    int unit = ONE && a.usage ? blockIdx.x * a.row_groups : blockIdx.x, t = 0, budget = 1 << 30, units = a.units;
    if constexpr (ONE) units = min(units, unit + (a.usage ? a.row_groups : 1));
    else {
        const bool some = find_begin<STEP>(a, unit, t, budget);
        if (threadIdx.x < 4) a.begins[blockIdx.x * 4 + threadIdx.x] = threadIdx.x == 0 ? (some ? unit : -1) : threadIdx.x == 1 ? t : budget;
        if (!some) return;
    }
    auto load = [&](const T *row) INLINE {      // this lane's 16 bytes; zeros behind the row's end
        if constexpr (WHOLE) {
            const AnyVec<T> v = load_any(row + min(d0, a.D - VEC));
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else return d0 < a.D ? load_run<T>(row + d0, a.D - d0) : make_uint4(0, 0, 0, 0);
    };
    for (; budget > 0 && unit < units; unit++, t = 0) {
        const int nh = unit / a.row_groups, row0 = (unit - nh * a.row_groups) * R, n = nh / a.heads, h = nh - n * a.heads;
        const int rows = min(R, a.group - row0), slots = slots_of(a, n), steps = max(1, (slots + STEP - 1) / STEP);
        const int t0 = t, t1 = ONE ? steps : min(steps, t + budget);
        budget -= t1 - t0;
        const T *kb = reinterpret_cast<const T *>(a.key) + h * a.ks[1], *vb = reinterpret_cast<const T *>(a.value) + h * a.vs[1];
        const int32_t *table = a.table + n * a.table_stride;
        float *scores = a.usage ? a.scores + (long)unit * a.slots_padded * R : nullptr;

        uint4 k[LOADS], v[LOADS];
        bool there[LOADS];
        int id[LOADS], in_page[LOADS];
        auto slot_of = [&](int step, int u) INLINE { return step * STEP + (u * 4 + wave) * KEYS + lane / LANES; };
        auto look = [&](int step) INLINE {
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const int s = min(slot_of(step, u), slots - 1), p = fdiv(s, a.page);
                id[u] = table[p];
                in_page[u] = s - p * a.page.d;
            }
        };
        auto request = [&](int step) INLINE {
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const bool valid = (unsigned)id[u] < (unsigned)a.pages;
                there[u] = valid && slot_of(step, u) < slots;
                const long page = valid ? id[u] : 0;
                k[u] = load(kb + page * a.ks[0] + in_page[u] * a.ks[2]);
                v[u] = load(vb + page * a.vs[0] + in_page[u] * a.vs[2]);
            }
        };
        if (slots > 0) {
            look(t);
            request(t);
            if (t + 1 < t1) look(t + 1);
        }
        uint4 q[R];
        float o[R][VEC], m[R], l[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const uint4 w = load(reinterpret_cast<const T *>(a.q) + n * a.qs[0] + (long)(h * a.group + row0 + min(r, rows - 1)) * a.qs[1]);
            q[r] = r < rows ? w : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < VEC; i++) o[r][i] = 0.f;
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
        for (; t < t1 && slots > 0; t++) {
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
            if (scores) {
                // (all lanes of a slot have its scores: lane u of them writes those of load u, all rows together)
                static_assert(LOADS <= LANES, "");
                float mine[R];
#pragma unroll
                for (int r = 0; r < R; r++) {
                    mine[r] = s[0][r];
#pragma unroll
                    for (int u = 1; u < LOADS; u++) mine[r] = lane % LANES == u ? s[u][r] : mine[r];
                }
                const int slot = slot_of(t, lane % LANES);
                if (lane % LANES < LOADS && slot < slots) {
#pragma unroll
                    for (int r = 0; r < R; r++) scores[(long)slot * R + r] = mine[r];
                }
            }
            if (t + 1 < t1) {
                request(t + 1);
                if (t + 2 < t1) look(t + 2);
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                float top = s[0][r];
#pragma unroll
                for (int u = 1; u < LOADS; u++) top = fmaxf(top, s[u][r]);
                // (the maximum follows where it has grown by more than a factor of 2^8 of the weights)
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
        t = t1;
        // the groups of lanes, two values to a step where half the wavefront can go on with either, then the wavefronts
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
        const bool direct = ONE || (t0 == 0 && t1 == steps);
        const long piece = ONE ? unit : (long)unit + blockIdx.x;
        for (int i = threadIdx.x; i < rows * DP; i += 256) {
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
            if (!ONE && d == 0) *reinterpret_cast<float2 *>(a.part_ml + (piece * R + r) * 2) = make_float2(top, sum);
            if (direct) reinterpret_cast<T *>(a.out)[((long)n * a.heads * a.group + h * a.group + row0 + r) * a.D + d] = f32_to_elem<T>(sum == 0.f ? 0.f : x / sum);
            else a.part[(piece * R + r) * part_width(a.D) + d] = x;
        }
        if (!ONE && threadIdx.x == 0) {
            if (t0 == 0) a.covered[unit * 2] = blockIdx.x;
            if (t1 == steps) a.covered[unit * 2 + 1] = blockIdx.x;
        }
        if constexpr (ONE) {
            if (a.usage) {
                if ((int)threadIdx.x < rows) {
                    const int r = threadIdx.x;
                    float top = s_ml[0][r].x, sum = 0.f;
#pragma unroll
                    for (int w = 1; w < 4; w++) top = fmaxf(top, s_ml[w][r].x);
                    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                    for (int w = 0; w < 4; w++) sum = fmaf(s_ml[w][r].y, __builtin_amdgcn_exp2f(s_ml[w][r].x - base), sum);
                    s_row[row0 + r] = usage_ml(top, sum);
                }
                __syncthreads();
                if (unit + 1 == units) add_usage<R, false>(a, unit + 1 - a.row_groups, n, h, 0, slots, s_row);
            }
        }
        __syncthreads();      // (s_o and s_ml are written again by the next unit's piece)
    }
}

// More than four rows of a key head, bfloat16: their products on the matrix instruction, whose columns are the rows (R of them, up to 32).  A wavefront has 32 slots of a step to
// itself, whose keys and values go through tiles of its own in LDS: neighbouring lanes ask for a whole slot's (pieces of 16 channels straight into the operand's place took 1.2 times as
// long where pages are scattered).  No barrier until the end of a unit's piece, where the four wavefronts' sums meet.  Weights are two terms, which cost little here.
// Bound: memory.
constexpr int kWideStep = 128;
template <int DP, bool WHOLE, int R, bool ONE> __global__ void __launch_bounds__(256, 2) mem_attn_wide_kernel(MemArgs a)
{
    typedef bf16_t T;
    using V = Tile<T, DP, 32, 64, WHOLE>;
    constexpr int ND = DP / 32, NK = DP / 16, LINE = DP + 1, SUMS = 4 * R * LINE * 4, TILES = 8 * V::BYTES, PER = V::PIECES / 2;
    __shared__ __align__(16) unsigned char s_mem[SUMS > TILES ? SUMS : TILES];
    __shared__ float2 s_ml[4][R], s_row[ONE ? 256 : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, row = lane & 31;
    unsigned char *s_k = s_mem + wave * 2 * V::BYTES, *s_v = s_k + V::BYTES;
    float *s_o = reinterpret_cast<float *>(s_mem);
    int unit = ONE && a.usage ? blockIdx.x * a.row_groups : blockIdx.x, t = 0, budget = 1 << 30, units = a.units;
    if constexpr (ONE) units = min(units, unit + (a.usage ? a.row_groups : 1));
    else {
        const bool some = find_begin<kWideStep>(a, unit, t, budget);
        if (threadIdx.x < 4) a.begins[blockIdx.x * 4 + threadIdx.x] = threadIdx.x == 0 ? (some ? unit : -1) : threadIdx.x == 1 ? t : budget;
        if (!some) return;
    }
    for (; budget > 0 && unit < units; unit++, t = 0) {
        const int nh = unit / a.row_groups, row0 = (unit - nh * a.row_groups) * R, n = nh / a.heads, h = nh - n * a.heads;
        const int rows = min(R, a.group - row0), slots = slots_of(a, n), steps = max(1, (slots + kWideStep - 1) / kWideStep);
        const int t0 = t, t1 = ONE ? steps : min(steps, t + budget);
        budget -= t1 - t0;
        const T *kb = reinterpret_cast<const T *>(a.key) + h * a.ks[1], *vb = reinterpret_cast<const T *>(a.value) + h * a.vs[1];
        const int32_t *table = a.table + n * a.table_stride;
        float *scores = a.usage ? a.scores + (long)unit * a.slots_padded * a.score_rows : nullptr;

        Raw8<T> k[PER], v[PER];
        bool there = false;
        int id = -1, in_page = 0;
        // lane % 32 knows the place of its slot of a step
        auto look = [&](int step) INLINE {
            const int s = min(step * kWideStep + wave * 32 + row, slots - 1), p = fdiv(s, a.page);
            id = table[p];
            in_page = s - p * a.page.d;
        };
        auto request = [&](int step) INLINE {
            there = (unsigned)id < (unsigned)a.pages && step * kWideStep + wave * 32 + row < slots;
            const int known = there ? id : -1;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int from = (i * 64 + lane) / V::PIECES, d = (i * 64 + lane) % V::PIECES * 8, page = __shfl(known, from, 64), at = __shfl(in_page, from, 64);
                k[i] = load8_of<WHOLE, T>(kb + max(page, 0) * a.ks[0] + at * a.ks[2], d, a.D, page >= 0);
                v[i] = load8_of<WHOLE, T>(vb + max(page, 0) * a.vs[0] + at * a.vs[2], d, a.D, page >= 0);
            }
        };
        if (slots > 0) {
            look(t);
            request(t);
            if (t + 1 < t1) look(t + 1);
        }
        Frag<1> q[NK];
        {
            const T *qr = reinterpret_cast<const T *>(a.q) + n * a.qs[0] + (long)(h * a.group + row0 + min(row, rows - 1)) * a.qs[1];
#pragma unroll
            for (int i = 0; i < NK; i++) q[i] = terms_of<T>(load8_of<WHOLE, T>(qr, i * 16 + half * 8, a.D, row < rows));
        }
        f32x16 o[ND];
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[i][r] = 0.f;
        float m = -INFINITY, lift = -INFINITY, l = 0.f;
        const float c = a.scale2;

        for (; t < t1 && slots > 0; t++) {
            const uint32_t some = (uint32_t)__ballot(there);
            f32x16 s;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = 0.f;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int at = piece_at<DP>((i * 64 + lane) / V::PIECES, (i * 64 + lane) % V::PIECES);
                *reinterpret_cast<uint4 *>(s_k + at) = k[i].v[0];
                *reinterpret_cast<uint4 *>(s_v + at) = v[i].v[0];
            }
#pragma unroll
            for (int i = 0; i < NK; i++) mma(s, V::rows(s_k, row, i, half), q[i]);
            if (t + 1 < t1) {
                request(t + 1);
                if (t + 2 < t1) look(t + 2);
            }
            if (some != 0xffffffffu) {
                const uint32_t b = some >> (half * 4);
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!((b >> (8 * (r / 4) + r % 4)) & 1)) s[r] = -INFINITY;
            }
            if (scores) {
                // (four neighbouring slots of a row at a time; what is behind the last of them is not read)
                if (row < rows && t * kWideStep + wave * 32 < slots) {
                    float *to = scores + row * a.slots_padded + t * kWideStep + wave * 32 + half * 4;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (t * kWideStep + wave * 32 + j * 8 < a.slots_padded)
                            *reinterpret_cast<float4 *>(to + j * 8) = make_float4(s[j * 4] * c, s[j * 4 + 1] * c, s[j * 4 + 2] * c, s[j * 4 + 3] * c);
                }
            }
            if (some == 0) continue;
            float top = s[0];
#pragma unroll
            for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
            // (the maximum follows where it has grown by more than a factor of 2^8 of the weights)
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
            float p[16];
#pragma unroll
            for (int r = 0; r < 16; r++) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -mc));
                l += p[r];
            }
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                const Frag<2> pf = make_frag<2, WEIGHTS>(p + kk * 8);
#pragma unroll
                for (int d = 0; d < ND; d++) mma(o[d], V::columns(s_v, kk * 16, d * 32, lane), pf);
            }
        }
        t = t1;
        l = half_sum(l);
        // the wavefronts' sums, in the place of their tiles
        if (half == 0 && row < R) s_ml[wave][row] = make_float2(m == -INFINITY ? -INFINITY : m * c, l);
        __syncthreads();
        if (row < rows) {
            float *to = s_o + (wave * R + row) * LINE;
#pragma unroll
            for (int i = 0; i < ND; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) to[i * 32 + 8 * (r / 4) + 4 * half + r % 4] = o[i][r];
        }
        __syncthreads();
        const bool direct = ONE || (t0 == 0 && t1 == steps);
        const long piece = ONE ? unit : (long)unit + blockIdx.x;
        for (int i = threadIdx.x; i < rows * DP; i += 256) {
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
                x = fmaf(s_o[(w * R + r) * LINE + d], f, x);
            }
            if (d == 0) {
                if constexpr (ONE) s_row[row0 + r] = usage_ml(top, sum);
                else *reinterpret_cast<float2 *>(a.part_ml + (piece * R + r) * 2) = make_float2(top, sum);
            }
            if (direct) reinterpret_cast<T *>(a.out)[((long)n * a.heads * a.group + h * a.group + row0 + r) * a.D + d] = f32_to_elem<T>(sum == 0.f ? 0.f : x / sum);
            else a.part[(piece * R + r) * part_width(a.D) + d] = x;
        }
        if (!ONE && threadIdx.x == 0) {
            if (t0 == 0) a.covered[unit * 2] = blockIdx.x;
            if (t1 == steps) a.covered[unit * 2 + 1] = blockIdx.x;
        }
        __syncthreads();      // (tiles and sums are written again by the next unit's piece)
        if constexpr (ONE) {
            if (a.usage && unit + 1 == units) add_usage<R, true>(a, unit + 1 - a.row_groups, n, h, 0, slots, s_row);
        }
    }
}

// Units that several workgroups have shared: blocks from 0, one to a row, put their pieces together.  Where weights are added up: blocks from `rows` on, kUsageBlocks to each
// workgroup of the walk, go over the same slots once more, by their scores.  Bound: the latency of its chain; 12.8 us where 32 streams' weights are added up (20 MB; 2 or 8 blocks to a
// workgroup, and requests before the rows' sums are known, are no shorter).
constexpr int kUsageBlocks = 4;
template <typename T, int LANES, int R, bool WIDE> __global__ void __launch_bounds__(256) mem_join_kernel(MemArgs a, int rows, int step)
{
    constexpr int GROUPS = 256 / LANES;
    __shared__ float4 s_x[256];
    __shared__ float2 s_ml[256];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < rows) {
        const int nh = blockIdx.x / a.group, row = blockIdx.x - nh * a.group, unit = nh * a.row_groups + row / R, r = row % R;
        const int w0 = a.covered[unit * 2], w1 = a.covered[unit * 2 + 1];
        if (w0 == w1) return;
        const int lane = tid % LANES, group = tid / LANES, d = lane * 4, width = part_width(a.D);
        float all = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int w = w0 + group; w <= w1; w += 4 * GROUPS) {
            float2 ml[4];
            float4 y[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const long from = (long)(unit + min(w + u * GROUPS, w1)) * R + r;
                ml[u] = *reinterpret_cast<const float2 *>(a.part_ml + from * 2);
                y[u] = *reinterpret_cast<const float4 *>(a.part + from * width + min(d, width - 4));
            }
            float top = all;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (w + u * GROUPS > w1) ml[u] = make_float2(-INFINITY, 0.f);
                top = fmaxf(top, ml[u].x);
            }
            const float base = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f(all - base);
            all = top;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] *= f;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (w + u * GROUPS > w1) continue;
                const float g = __builtin_amdgcn_exp2f(ml[u].x - base);
                l = fmaf(ml[u].y, g, l);
                x[0] = fmaf(y[u].x, g, x[0]); x[1] = fmaf(y[u].y, g, x[1]); x[2] = fmaf(y[u].z, g, x[2]); x[3] = fmaf(y[u].w, g, x[3]);
            }
        }
        s_x[tid] = make_float4(x[0], x[1], x[2], x[3]);
        s_ml[tid] = make_float2(all, l);
        __syncthreads();
        if (group != 0) return;
        const int some = min(GROUPS, w1 - w0 + 1);
        for (int g = 1; g < some; g++) all = fmaxf(all, s_ml[g * LANES].x);
        const float base = all == -INFINITY ? 0.f : all;
        l = x[0] = x[1] = x[2] = x[3] = 0.f;
        for (int g = 0; g < some; g++) {
            const float2 ml = s_ml[g * LANES];
            const float4 y = s_x[tid + g * LANES];
            const float f = __builtin_amdgcn_exp2f(ml.x - base);
            l = fmaf(ml.y, f, l);
            x[0] = fmaf(y.x, f, x[0]); x[1] = fmaf(y.y, f, x[1]); x[2] = fmaf(y.z, f, x[2]); x[3] = fmaf(y.w, f, x[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = l == 0.f ? 0.f : x[i] / l;
        if (d < a.D) store4<T>(reinterpret_cast<T *>(a.out) + ((long)nh * a.group + row) * a.D + d, x, a.D - d);
        return;
    }
    const int32_t *begin = a.begins + ((int)blockIdx.x - rows) / kUsageBlocks * 4;
    int unit = begin[0], t = begin[1], budget = begin[2];
    if (unit < 0) return;
    const int part = ((int)blockIdx.x - rows) % kUsageBlocks;
    for (; budget > 0 && unit < a.units; unit++, t = 0) {
        const int nh = unit / a.row_groups, n = nh / a.heads, h = nh - n * a.heads, slots = slots_of(a, n), steps = max(1, (slots + step - 1) / step);
        const int t1 = min(steps, t + budget);
        budget -= t1 - t;
        if (unit != nh * a.row_groups || slots == 0) continue;      // (the first group of rows goes for all of them)
        const int s0 = t * step, some = min(slots, t1 * step) - s0, from = s0 + (int)((long)some * part / kUsageBlocks), to = s0 + (int)((long)some * (part + 1) / kUsageBlocks);
        if (from == to) continue;
        __syncthreads();
        for (int row = tid >> 6; row < a.group; row += 4) {
            const int u = unit + row / R, w0 = a.covered[u * 2], w1 = a.covered[u * 2 + 1];
            float top = -INFINITY, sum = 0.f;
            for (int w = w0 + (tid & 63); w <= w1; w += 64) {
                const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + ((long)(u + w) * R + row % R) * 2);
                const float grown = fmaxf(top, ml.x), base = grown == -INFINITY ? 0.f : grown;
                sum = sum * __builtin_amdgcn_exp2f(top - base) + ml.y * __builtin_amdgcn_exp2f(ml.x - base);
                top = grown;
            }
            float all = top;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) all = fmaxf(all, __shfl_xor(all, d, 64));
            sum *= __builtin_amdgcn_exp2f(top - (all == -INFINITY ? 0.f : all));
            sum = lanes_sum<64>(sum);
            if ((tid & 63) == 0) s_ml[row] = usage_ml(all, sum);
        }
        __syncthreads();
        add_usage<R, WIDE>(a, unit, n, h, from, to, s_ml);
    }
}

// ---------------------------------------------------------------- append
struct AppendArgs {
    const void *nk, *nv;
    void *key, *value;
    const int32_t *table, *starts;      // starts: or NULL
    int32_t *lengths, *seen, *positions;
    float *usage;
    long nks[2], nvs[2], ks[3], vs[3], table_stride, tokens;
    FastDiv page;
    int N, heads, D, pages, slots;
};
D2C_DEV long start_of(const AppendArgs &a, int n) { return min(max((long)a.starts[n], 0L), a.tokens); }

// One new token of one stream's head: its key and value by pieces of 16 bytes, its usage and position
template <typename T> D2C_DEV void put_piece(const AppendArgs &a, long token, int n, long slot, int position, int h, int piece, int pieces)
{
    if (slot >= a.slots) return;
    const int p = fdiv((int)slot, a.page), id = a.table[n * a.table_stride + p], at = (int)slot - p * a.page.d;
    if ((unsigned)id >= (unsigned)a.pages) return;
    constexpr int VEC = 16 / (int)sizeof(T);
    const bool second = piece >= pieces;
    const int d = (second ? piece - pieces : piece) * VEC;
    const T *from = second ? reinterpret_cast<const T *>(a.nv) + token * a.nvs[0] + h * a.nvs[1] : reinterpret_cast<const T *>(a.nk) + token * a.nks[0] + h * a.nks[1];
    T *to = second ? reinterpret_cast<T *>(a.value) + id * a.vs[0] + h * a.vs[1] + at * a.vs[2] : reinterpret_cast<T *>(a.key) + id * a.ks[0] + h * a.ks[1] + at * a.ks[2];
    store_run<T>(to + d, load_run<T>(from + d, a.D - d), a.D - d);
    if (piece == 0) {
        const long i = ((long)id * a.heads + h) * a.page.d + at;
        a.usage[i] = 0.f;
        a.positions[i] = position;
    }
}
// A token of each stream: a workgroup to a stream, which then lets its counts grow.  One launch; latency: 64 streams of 4 heads of 64, 3.0 us.
template <typename T> __global__ void __launch_bounds__(256) mem_append_one_kernel(AppendArgs a)
{
    const int n = blockIdx.x, pieces = (a.D * (int)sizeof(T) + 15) / 16, all = a.heads * pieces * 2;
    const int length = min(max(a.lengths[n], 0), a.slots), seen = a.seen[n];
    for (int i = threadIdx.x; i < all; i += 256) put_piece<T>(a, n, n, length, seen, i / (pieces * 2), i % (pieces * 2), pieces);
    __syncthreads();
    if (threadIdx.x == 0) {
        a.lengths[n] = min(length + 1, a.slots);
        a.seen[n] = seen + 1;
    }
}
// Packed tokens, kAppendTokens to a workgroup: a thread to a token finds its place, then all of them move pieces of 16 bytes, four requested at a time.  Bound: memory; four clips of up to 12960
// tokens, 8 heads of 64, bfloat16, 21 us (93 MB, 4.4 TB/s).
constexpr int kAppendTokens = 8;
template <typename T> __global__ void __launch_bounds__(256) mem_append_kernel(AppendArgs a, FastDiv by_pieces)
{
    constexpr int VEC = 16 / (int)sizeof(T), AT_ONCE = 4;
    __shared__ int s_page[kAppendTokens], s_slot[kAppendTokens];      // (page -1: nowhere)
    const long token0 = (long)blockIdx.x * kAppendTokens;
    const int tid = threadIdx.x;
    if (tid < kAppendTokens) {
        int id = -1, at = 0;
        const long token = token0 + tid;
        if (token < a.tokens) {
            int lo = 0, hi = a.N;      // the last stream that begins at or before the token
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start_of(a, mid) <= token) lo = mid; else hi = mid;
            }
            const long first = start_of(a, lo), slot = min(max(a.lengths[lo], 0), a.slots) + token - first;
            if (token >= first && token < start_of(a, lo + 1) && slot < a.slots) {
                const int p = fdiv((int)slot, a.page);
                id = a.table[lo * a.table_stride + p];
                at = (int)slot - p * a.page.d;
                if ((unsigned)id >= (unsigned)a.pages) id = -1;
                else
                    for (int h = 0; h < a.heads; h++) {
                        const long i = ((long)id * a.heads + h) * a.page.d + at;
                        a.usage[i] = 0.f;
                        a.positions[i] = (int)(a.seen[lo] + token - first);
                    }
            }
        }
        s_page[tid] = id;
        s_slot[tid] = at;
    }
    __syncthreads();
    const int pieces = by_pieces.d, all = kAppendTokens * a.heads * pieces;      // (of keys; the same again of values)
    for (int i0 = tid; i0 < 2 * all; i0 += 256 * AT_ONCE) {
        T *to[AT_ONCE];
        uint4 x[AT_ONCE];
        int left[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            to[u] = nullptr;
            int i = i0 + u * 256;
            if (i >= 2 * all) continue;
            const bool second = i >= all;
            if (second) i -= all;
            const int row = fdiv(i, by_pieces), d = (i - row * pieces) * VEC, which = row / a.heads, h = row - which * a.heads, id = s_page[which];
            if (id < 0) continue;
            left[u] = a.D - d;
            const T *from = second ? reinterpret_cast<const T *>(a.nv) + (token0 + which) * a.nvs[0] + h * a.nvs[1]
                                   : reinterpret_cast<const T *>(a.nk) + (token0 + which) * a.nks[0] + h * a.nks[1];
            to[u] = d + (second ? reinterpret_cast<T *>(a.value) + id * a.vs[0] + h * a.vs[1] + s_slot[which] * a.vs[2]
                                : reinterpret_cast<T *>(a.key) + id * a.ks[0] + h * a.ks[1] + s_slot[which] * a.ks[2]);
            x[u] = load_run<T>(from + d, left[u]);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
            if (to[u]) store_run<T>(to[u], x[u], left[u]);
    }
}
__global__ void __launch_bounds__(256) mem_count_kernel(AppendArgs a)
{
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= a.N) return;
    const long some = max(start_of(a, n + 1) - start_of(a, n), 0L);
    a.lengths[n] = (int)min((long)min(max(a.lengths[n], 0), a.slots) + some, (long)a.slots);
    a.seen[n] = (int)(a.seen[n] + some);
}

// ---------------------------------------------------------------- evict
struct EvictArgs {
    void *key, *value;
    const int32_t *table, *seen;
    int32_t *lengths, *positions;
    float *usage;
    uint32_t *ranks;             // [units][slots_padded]
    int32_t *holes, *fillers;    // [units][pairs]
    int32_t *counts;             // [units]
    long ks[3], vs[3], table_stride, slots_padded;
    FastDiv page;
    int N, heads, D, pages, slots, keep, recent, pairs;
};

// What a slot is ranked by: usage as a number that sorts like it (NaN above all), above it what is to stay whatever its usage, below it what is not there
D2C_DEV uint32_t rank_of(float usage, bool stays)
{
    if (stays) return 0xffffffffu;
    if (usage != usage) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(usage + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A workgroup to a stream's head.  The keep-th largest rank by its digits (11, 11 and 10 bits, a histogram of each in LDS, the first in several copies, whose few bins many
// lanes meet in), then the slots that go before `keep` and those that stay behind it, each in rising order.  A wavefront has neighbouring slots, 64 at a time, whose
// truth values are one word each: counted by a lane to a word.
// Bound: a compute unit's instructions and the latency of its chain (counts, pages, usage, three histograms).  64 units of up to 25920 slots 35 us (33 with the ranks in LDS, as far as they have
// room there; 44 with a request for each page after the other; 51 with ranks in registers and loops unrolled, whose instructions every launch fetches anew), 4 units of 3240 slots 10.5.  Where all
// usages are equal (a memory that was read without them being added up) lanes wait for one bin and one count: whole passes, 64 units of up to 25920 slots 100 us instead of 72, one of 64800 191
// instead of 75.
constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;
__global__ void __launch_bounds__(kEvictThreads) mem_rank_kernel(EvictArgs a)
{
    constexpr int BINS = 2048, COPIES = 4, AT_ONCE = 4, WORDS = 64;
    constexpr int LIST = (COPIES - 1) * BINS, REQUESTS = 8;
    __shared__ __align__(16) int s_hist[COPIES][BINS];
    __shared__ __align__(16) uint4 s_words[kEvictWaves][WORDS];      // of 64 slots: which ranks are above the border, which are at it
    __shared__ int s_wave[3][kEvictWaves], s_digit[2], s_met;
    const int unit = blockIdx.x, n = unit / a.heads, h = unit - n * a.heads, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slots = min(max(a.lengths[n], 0), a.slots);
    if (slots <= a.keep || a.pages == 0) {      // (without pages there is nothing to rank, nor to read)
        if (tid == 0) a.counts[unit] = 0;
        return;
    }
    const int per = (slots + kEvictThreads - 1) / kEvictThreads * 64, s0 = min(wave * per, slots), s1 = min(s0 + per, slots), numbers = (s1 - s0 + 63) / 64;
    const int newest = (int)max((long)a.seen[n] - a.recent, -(1L << 31));
    const int32_t *table = a.table + n * a.table_stride;
    uint32_t *ranks = a.ranks + unit * a.slots_padded;
    uint32_t *s_list = reinterpret_cast<uint32_t *>(s_hist[1]);      // ranks of the second pass's digit, in the place of the first pass's copies
    // f(number, rank) for the wavefront's slots s0 + 64 number + lane from number `first` on, 4 at a time and WORDS at most
    auto for_slots = [&](int first, auto f) INLINE {
#pragma unroll 1
        for (int i = first; i < min(numbers, first + WORDS); i += AT_ONCE) {
            uint32_t r[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                const int s = s0 + (i + u) * 64 + lane;
                r[u] = ranks[min(s, s1 - 1)];
                if (s >= s1) r[u] = 0;
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) f(i + u, r[u]);
        }
    };
    if (tid == 0) s_met = 0;
    for (int i = tid; i < COPIES * BINS / 4; i += kEvictThreads) reinterpret_cast<int4 *>(&s_hist[0][0])[i] = make_int4(0, 0, 0, 0);
    // ranks, REQUESTS numbers at a time; 0 for what is not there
#pragma unroll 1
    for (int i = 0; i < numbers; i += REQUESTS) {
        int id[REQUESTS], in_page[REQUESTS], positions[REQUESTS];
        float usage[REQUESTS];
#pragma unroll
        for (int u = 0; u < REQUESTS; u++) {
            const int s = min(s0 + (i + u) * 64 + lane, slots - 1), p = fdiv(s, a.page);
            id[u] = table[p];
            in_page[u] = s - p * a.page.d;
        }
#pragma unroll
        for (int u = 0; u < REQUESTS; u++) {
            const long at = ((long)((unsigned)id[u] < (unsigned)a.pages ? id[u] : 0) * a.heads + h) * a.page.d + in_page[u];
            usage[u] = a.usage[at];
            positions[u] = a.positions[at];
        }
#pragma unroll
        for (int u = 0; u < REQUESTS; u++) {
            const int s = s0 + (i + u) * 64 + lane;
            const uint32_t rank = (unsigned)id[u] < (unsigned)a.pages ? rank_of(usage[u], positions[u] >= newest) : 0u;
            if (s < s1) ranks[s] = rank;
        }
    }
    uint32_t prefix = 0;
    int wanted = a.keep;
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        if (pass > 0)
            for (int i = tid; i < BINS / 4; i += kEvictThreads) reinterpret_cast<int4 *>(s_hist[0])[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
        if (pass == 0)
            for (int first = 0; first < numbers; first += WORDS)
                for_slots(first, [&](int, uint32_t rank) INLINE {
                    if (rank != 0) atomicAdd(&s_hist[lane % COPIES][rank >> 21], 1);
                });
        else if (pass == 1)
            for (int first = 0; first < numbers; first += WORDS)
                for_slots(first, [&](int, uint32_t rank) INLINE {
                    if ((rank >> 21) != (prefix >> 21)) return;
                    atomicAdd(&s_hist[0][(rank >> 10) & 2047], 1);
                    const int at = atomicAdd(&s_met, 1);      // (in any order: they are only counted)
                    if (at < LIST) s_list[at] = rank;
                });
        else if (s_met <= LIST)
            for (int i = tid; i < s_met; i += kEvictThreads) {
                if ((s_list[i] >> 10) == (prefix >> 10)) atomicAdd(&s_hist[0][s_list[i] & 1023], 1);
            }
        else
            for (int first = 0; first < numbers; first += WORDS)
                for_slots(first, [&](int, uint32_t rank) INLINE {
                    if ((rank >> 10) == (prefix >> 10)) atomicAdd(&s_hist[0][rank & 1023], 1);
                });
        __syncthreads();
        // bins from the top: thread i has bins 2047 - 2i and 2046 - 2i
        int high = 0, low = 0;
#pragma unroll 1
        for (int c = 0; c < (pass == 0 ? COPIES : 1); c++) {
            const int2 two = *reinterpret_cast<const int2 *>(&s_hist[c][BINS - 2 - 2 * tid]);
            high += two.y; low += two.x;
        }
        // (slots of rank 0 are counted nowhere: where others do not make up `keep`, the last bin has what is wanted)
        if (tid == kEvictThreads - 1) low = a.slots;
        const int scan = wave_scan(high + low);
        if (lane == 63) s_wave[0][wave] = scan;
        __syncthreads();
        const int above = scan - high - low + before_wave<kEvictWaves>(s_wave[0], wave);
        if (above < wanted && wanted <= above + high) { s_digit[0] = BINS - 1 - 2 * tid; s_digit[1] = wanted - above; }
        else if (above + high < wanted && wanted <= above + high + low) { s_digit[0] = BINS - 2 - 2 * tid; s_digit[1] = wanted - above - high; }
        __syncthreads();
        prefix |= (uint32_t)s_digit[0] << shift;
        wanted = s_digit[1];      // how many of this digit stay, in the end: of the rank itself, lowest slots first
    }
    // lane i has the words of number first + i
    uint64_t above = 0, same = 0;
    auto find_words = [&](int first) INLINE {
        for_slots(first, [&](int i, uint32_t rank) INLINE {
            const uint64_t x = __ballot(rank > prefix), y = __ballot(rank == prefix);
            s_words[wave][i - first] = make_uint4((uint32_t)x, (uint32_t)(x >> 32), (uint32_t)y, (uint32_t)(y >> 32));      // (all lanes the same)
        });
        __builtin_amdgcn_wave_barrier();
        const uint4 w = s_words[wave][min(lane, WORDS - 1)];
        // (slots behind the last have a rank of 0, which may be the border)
        const int s = s0 + (first + lane) * 64;
        const uint64_t live = s >= s1 || lane >= WORDS ? 0 : s1 - s >= 64 ? ~0ull : (1ull << (s1 - s)) - 1;
        above = live & ((uint64_t)w.x | (uint64_t)w.y << 32);
        same = live & ((uint64_t)w.z | (uint64_t)w.w << 32);
        return live;
    };
    int equal = 0;
    for (int first = 0; first < numbers; first += WORDS) {
        find_words(first);
        equal += __builtin_amdgcn_readlane(wave_scan(__popcll(same)), 63);
    }
    if (lane == 0) s_wave[0][wave] = equal;
    __syncthreads();
    const int ties = before_wave<kEvictWaves>(s_wave[0], wave);
    // of this lane's words: slots that go before `keep`, slots that stay behind it
    int seen = ties;
    uint64_t hole = 0, filler = 0;
    auto sort_out = [&](int first) INLINE {
        const uint64_t live = find_words(first);
        const int count = __popcll(same), scan = wave_scan(count);
        int left = min(max(wanted - (seen + scan - count), 0), count);      // of the ties: the first so many stay
        seen += __builtin_amdgcn_readlane(scan, 63);
        uint64_t stays = above, rest = same;
        if (left == count) stays |= same;
        else
            for (; left > 0; left--) { stays |= rest & -rest; rest &= rest - 1; }
        const int s = s0 + (first + lane) * 64;
        const uint64_t low = s >= a.keep ? 0 : a.keep - s >= 64 ? ~0ull : (1ull << (a.keep - s)) - 1;
        hole = live & ~stays & low;
        filler = stays & ~low;
    };
    int holes = 0, fillers = 0;
    for (int first = 0; first < numbers; first += WORDS) {
        sort_out(first);
        holes += __builtin_amdgcn_readlane(wave_scan(__popcll(hole)), 63);
        fillers += __builtin_amdgcn_readlane(wave_scan(__popcll(filler)), 63);
    }
    if (lane == 0) { s_wave[1][wave] = holes; s_wave[2][wave] = fillers; }
    __syncthreads();
    holes = before_wave<kEvictWaves>(s_wave[1], wave);
    fillers = before_wave<kEvictWaves>(s_wave[2], wave);
    seen = ties;
    int32_t *to = a.holes + (long)unit * a.pairs, *of = a.fillers + (long)unit * a.pairs;
    for (int first = 0; first < numbers; first += WORDS) {
        if (numbers > WORDS) sort_out(first);
        const int h1 = wave_scan(__popcll(hole)), f1 = wave_scan(__popcll(filler)), h0 = holes + h1 - __popcll(hole), f0 = fillers + f1 - __popcll(filler);
        auto put = [&](int32_t *list, uint64_t mine, int base, int i, int slot) INLINE {
            const uint32_t lo = __builtin_amdgcn_readlane((int)mine, i), hi = __builtin_amdgcn_readlane((int)(mine >> 32), i);
            const unsigned at = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, __builtin_amdgcn_readlane(base, i)));
            if (__builtin_amdgcn_inverse_ballot_w64((uint64_t)lo | (uint64_t)hi << 32)) list[at] = slot;
        };
        for (int i = 0; i < min(numbers - first, WORDS); i++) {
            const int s = s0 + (first + i) * 64;
            if (s < a.keep) put(to, hole, h0, i, s + lane);
            if (s + 64 > a.keep) put(of, filler, f0, i, s + lane);
        }
        holes += __builtin_amdgcn_readlane(h1, 63);
        fillers += __builtin_amdgcn_readlane(f1, 63);
    }
    if (wave == kEvictWaves - 1 && lane == 0) a.counts[unit] = holes;
}
// What stays behind `keep` into the places of what goes before it: reads and writes meet nowhere.  kMovePairs to a workgroup: a thread to a pair finds both places and
// moves usage and position, then all of them move pieces of 16 bytes, four requested at a time.  Bound: memory, rows of 128 bytes here and there; eight streams of 8 heads of 64, bfloat16, 36 us
// (145 MB, 4.0 TB/s; 44 with both places looked up for every piece).
constexpr int kMovePairs = 64;
template <typename T> __global__ void __launch_bounds__(256) mem_move_kernel(EvictArgs a, int blocks, FastDiv by_pieces)
{
    constexpr int VEC = 16 / (int)sizeof(T), AT_ONCE = 4;
    __shared__ int s_to[kMovePairs][2], s_of[kMovePairs][2];      // page (-1: nowhere) and place
    const int unit = blockIdx.x / blocks, block = blockIdx.x - unit * blocks, n = unit / a.heads, h = unit - n * a.heads, count = a.counts[unit], tid = threadIdx.x;
    if (block == 0 && h == 0 && tid == 0) a.lengths[n] = min(min(max(a.lengths[n], 0), a.slots), a.keep);
    const int32_t *table = a.table + n * a.table_stride;
    for (int first = block * kMovePairs; first < count; first += blocks * kMovePairs) {
        const int some = min(kMovePairs, count - first);
        if (tid < some) {
            const int hole = a.holes[(long)unit * a.pairs + first + tid], filler = a.fillers[(long)unit * a.pairs + first + tid];
            const int tp = fdiv(hole, a.page), fp = fdiv(filler, a.page), td = table[tp], fd = table[fp], ti = hole - tp * a.page.d, fi = filler - fp * a.page.d;
            const bool valid = (unsigned)td < (unsigned)a.pages && (unsigned)fd < (unsigned)a.pages;
            s_to[tid][0] = valid ? td : -1; s_to[tid][1] = ti;
            s_of[tid][0] = fd; s_of[tid][1] = fi;
            if (valid) {
                const long to = ((long)td * a.heads + h) * a.page.d + ti, of = ((long)fd * a.heads + h) * a.page.d + fi;
                a.usage[to] = a.usage[of];
                a.positions[to] = a.positions[of];
            }
        }
        __syncthreads();
        const int pieces = by_pieces.d, all = some * pieces;      // (of keys; the same again of values)
        for (int i0 = tid; i0 < 2 * all; i0 += 256 * AT_ONCE) {
            T *to[AT_ONCE];
            uint4 x[AT_ONCE];
            int left[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                to[u] = nullptr;
                int i = i0 + u * 256;
                if (i >= 2 * all) continue;
                const bool second = i >= all;
                if (second) i -= all;
                const int pair = fdiv(i, by_pieces), d = (i - pair * pieces) * VEC, page = s_to[pair][0];
                if (page < 0) continue;
                T *base = reinterpret_cast<T *>(second ? a.value : a.key) + h * (second ? a.vs[1] : a.ks[1]) + d;
                const long ps = second ? a.vs[0] : a.ks[0], ss = second ? a.vs[2] : a.ks[2];
                left[u] = a.D - d;
                to[u] = base + page * ps + s_to[pair][1] * ss;
                x[u] = load_run<T>(base + s_of[pair][0] * ps + s_of[pair][1] * ss, left[u]);
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++)
                if (to[u]) store_run<T>(to[u], x[u], left[u]);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side
int check(const d2c_memory_desc *q)
{
    if (!q) { d2c_set_error("memory: null description"); return D2C_ERR_SHAPE; }
    if (q->dtype != D2C_F32 && q->dtype != D2C_BF16) { d2c_set_error("memory: float32 or bfloat16 only"); return D2C_ERR_DTYPE; }
    if (q->streams < 0 || q->pages < 0 || q->per_stream < 0 || q->heads <= 0 || q->D <= 0 || q->page <= 0) {
        d2c_set_error("memory: sizes must not be negative, heads, their size and the page's positive");
        return D2C_ERR_SHAPE;
    }
    if (q->D > 128) { d2c_set_error("memory: heads of up to 128 channels, got %d", q->D); return D2C_ERR_UNSUPPORTED; }
    // (slots of a stream, steps of all and a launch's threads are counted in 32 bits)
    if ((long)q->per_stream * q->page >= (1L << 30) || (long)q->streams * q->heads >= (1L << 21) || q->streams >= (1 << 20)) {
        d2c_set_error("memory: too many streams, heads or slots");
        return D2C_ERR_SHAPE;
    }
    return D2C_OK;
}
int check(const d2c_memory_desc *q, const d2c_memory_query_desc *x)
{
    if (int rc = check(q)) return rc;
    if (!x) { d2c_set_error("memory_attention: null description"); return D2C_ERR_SHAPE; }
    if (x->query_heads <= 0 || x->query_heads % q->heads != 0) {
        d2c_set_error("memory_attention: %d query heads are no positive multiple of %d key heads", x->query_heads, q->heads);
        return D2C_ERR_SHAPE;
    }
    if (x->query_heads / q->heads > 256) { d2c_set_error("memory_attention: up to 256 query heads to a key head"); return D2C_ERR_UNSUPPORTED; }
    if (!(x->scale > 0.f) || !(x->scale < INFINITY)) { d2c_set_error("memory_attention: scale must be positive and finite"); return D2C_ERR_SHAPE; }
    const long slots = (long)q->per_stream * q->page;
    if ((long)q->streams * x->query_heads >= (1L << 23) || (long)q->streams * x->query_heads * (slots / 32 + 1) >= (1L << 30)) { d2c_set_error("memory_attention: too many streams, heads or slots"); return D2C_ERR_SHAPE; }
    return D2C_OK;
}
int need(const void *ws, size_t have, size_t bytes)
{
    if (!bytes || (ws && have >= bytes && !((uintptr_t)ws & 255u))) return D2C_OK;
    d2c_set_error("workspace of %zu bytes (256-byte aligned) required, got %zu at %p", bytes, have, ws);
    return D2C_ERR_WORKSPACE;
}

// f(T, LANES, R) as constants
template <typename F> auto for_rows(const d2c_memory_desc &q, int group, F f)
{
    auto with_type = [&](auto zero) {
        using T = decltype(zero);
        constexpr int L32 = 32 * (int)sizeof(T) / 16;
        auto with_lanes = [&](auto lanes) {
            if (group <= 1) return f(zero, lanes, std::integral_constant<int, 1>{});
            if (group <= 2) return f(zero, lanes, std::integral_constant<int, 2>{});
            if (group <= 4) return f(zero, lanes, std::integral_constant<int, 4>{});
            return f(zero, lanes, std::integral_constant<int, 8>{});
        };
        if (q.D <= 32) return with_lanes(std::integral_constant<int, L32>{});
        if (q.D <= 64) return with_lanes(std::integral_constant<int, 2 * L32>{});
        return with_lanes(std::integral_constant<int, 4 * L32>{});
    };
    return q.dtype == D2C_BF16 ? with_type(bf16_t{}) : with_type(float{});
}

// Memories of up to so many steps (of 32 to 256 slots) are read by a workgroup to each unit, in one launch: 8 heads of 64, bfloat16, 512 slots of 1 stream 6.9 us (else 9.3), 1024
// 10.5 (8.9); of 64 streams, whose units fill the GPU, 1024 21.7 (24.3)
constexpr int kOneSteps = 4, kOneStepsMany = 8;
// bfloat16 calls of more rows to a key head run on the matrix instruction (four rows, 64 channels, 32 streams of up to 12960 slots with weights added up: 77 us by lanes, 80 there; five
// rows, 64 streams of 4096: 19 there; 12 rows, 46 streams of 4096, 96 channels: 424 by lanes, 118 there)
constexpr int kTokenRows = 4;
struct MemPlan { int rows, score_rows, step, row_groups, units, places, least; bool wide, one; size_t part_bytes, ml_bytes, covered_bytes, begins_bytes, scores_bytes, bytes; long slots_padded; };
MemPlan mem_plan(const d2c_memory_desc &q, const d2c_memory_query_desc &x, bool track)
{
    MemPlan p{};
    const int group = x.query_heads / q.heads;
    p.wide = q.dtype == D2C_BF16 && group > kTokenRows;
    if (p.wide) { p.rows = group <= 16 ? 16 : 32; p.step = kWideStep; p.score_rows = std::min(group, p.rows); }
    else for_rows(q, group, [&](auto zero, auto lanes, auto r) {
        p.rows = p.score_rows = decltype(r)::value;
        p.step = TokenShape<decltype(zero), decltype(lanes)::value, decltype(r)::value>::STEP;
        return 0;
    });
    const long slots = (long)q.per_stream * q.page;
    p.row_groups = (group + p.rows - 1) / p.rows;
    p.units = q.streams * q.heads * p.row_groups;
    p.places = 2 * std::max(d2c_num_cus(), 1);
    p.least = 2;
    p.one = slots <= (long)(p.units >= p.places ? kOneStepsMany : kOneSteps) * p.step;
    p.slots_padded = (slots + 63) / 64 * 64;
    if (track) p.scores_bytes = d2c_align_up((size_t)p.units * p.score_rows * p.slots_padded * 4);
    if (!p.one) {
        const size_t lines = ((size_t)p.units + p.places) * p.rows;
        p.part_bytes = d2c_align_up(lines * part_width(q.D) * 4);
        p.ml_bytes = d2c_align_up(lines * 8);
        p.covered_bytes = d2c_align_up((size_t)p.units * 8);
        p.begins_bytes = d2c_align_up((size_t)p.places * 16);
    }
    p.bytes = p.part_bytes + p.ml_bytes + p.covered_bytes + p.begins_bytes + p.scores_bytes;
    return p;
}

// A call's streams, as many at a time as the limit has room for what goes by their slots, `bytes` of each: tables may have room for many times what streams hold, and lengths are not known here.
// All parts but the last have the same number.
inline int streams_at_once(int streams, size_t bytes, size_t limit)
{
    const long most = std::max((long)(limit / std::max(bytes, (size_t)1)), 1L), parts = (streams + most - 1) / most;
    return parts <= 1 ? streams : (int)((streams + parts - 1) / parts);
}
inline d2c_memory_desc with_streams(d2c_memory_desc q, int streams) { q.streams = streams; return q; }
// f(first stream, description of a part): the first result that is not D2C_OK
template <typename F> int for_streams(const d2c_memory_desc &q, int at_once, F f)
{
    for (int n = 0; n < q.streams; n += at_once)
        if (int rc = f(n, with_streams(q, std::min(at_once, q.streams - n)))) return rc;
    return D2C_OK;
}
// Scores of a tracked call: as the partial sums of attention, 256 MB at most (64 streams with room for 129600 tokens, 48 query heads: 1.6 GB otherwise)
int attention_streams(const d2c_memory_desc &q, const d2c_memory_query_desc &x, bool track)
{
    return track ? streams_at_once(q.streams, mem_plan(with_streams(q, 1), x, true).scores_bytes, D2C_ATTENTION_PART_BYTES) : q.streams;
}

struct EvictPlan { int pairs; long slots_padded; size_t ranks_bytes, list_bytes, bytes; };
EvictPlan evict_plan(const d2c_memory_desc &q, int keep)
{
    EvictPlan p{};
    const long slots = (long)q.per_stream * q.page;
    const size_t units = (size_t)q.streams * q.heads;
    if (slots <= keep || units == 0) return p;
    p.pairs = (int)std::min((long)keep, slots - keep);
    p.slots_padded = (slots + 63) / 64 * 64;
    p.ranks_bytes = d2c_align_up(units * p.slots_padded * 4);
    p.list_bytes = d2c_align_up(units * p.pairs * 4);
    p.bytes = p.ranks_bytes + 2 * p.list_bytes + d2c_align_up(units * 4);
    return p;
}
// Ranks and places: 1 GB at most.  (They are ranked by a workgroup to a stream's head, so that a limit which leaves compute units empty would cost time: two workgroups to each, of streams of
// 129600 slots, take 0.5 GB)
constexpr size_t kEvictBytes = (size_t)1 << 30;
int evict_streams(const d2c_memory_desc &q, int keep) { return streams_at_once(q.streams, evict_plan(with_streams(q, 1), keep).bytes, kEvictBytes); }

// Streams whose scores have room at once
int attend(const d2c_memory_desc *q, const d2c_memory_query_desc *x, const void *query, const void *key, const void *value, const int32_t *table, const int32_t *lengths, float *usage, void *out,
           void *ws, size_t ws_bytes, hipStream_t st)
{
    const long slots = (long)q->per_stream * q->page;
    const MemPlan p = mem_plan(*q, *x, usage != nullptr);
    if (int rc = need(ws, ws_bytes, p.bytes)) return rc;
    MemArgs a{};
    a.q = query; a.key = const_cast<void *>(key); a.value = const_cast<void *>(value); a.out = out; a.table = table; a.lengths = lengths; a.usage = usage;
    char *w = (char *)ws;
    a.part = (float *)w; a.part_ml = (float *)(w + p.part_bytes); a.covered = (int32_t *)(w + p.part_bytes + p.ml_bytes);
    a.begins = (int32_t *)(w + p.part_bytes + p.ml_bytes + p.covered_bytes);
    a.scores = (float *)(w + p.part_bytes + p.ml_bytes + p.covered_bytes + p.begins_bytes);
    for (int i = 0; i < 2; i++) a.qs[i] = x->query_stride[i];
    for (int i = 0; i < 3; i++) { a.ks[i] = q->key_stride[i]; a.vs[i] = q->value_stride[i]; }
    a.table_stride = q->table_stride; a.slots_padded = p.slots_padded; a.page = make_fastdiv(q->page);
    a.N = q->streams; a.heads = q->heads; a.group = x->query_heads / q->heads; a.D = q->D; a.pages = q->pages;
    a.slots = q->pages > 0 ? (int)slots : 0;      // (without pages no slot is there)
    a.score_rows = p.score_rows; a.row_groups = p.row_groups; a.units = p.units; a.places = p.places; a.least = p.least;
    a.scale2 = x->scale * 1.44269504088896340736f;
    const bool whole = q->D * d2c_elem_size(q->dtype) % 16 == 0;
    const dim3 grid(p.one ? (usage ? p.units / p.row_groups : p.units) : p.places), joins((unsigned)(q->streams * x->query_heads + (usage ? p.places * kUsageBlocks : 0)));
    auto join = [&](auto zero, auto lanes, auto r) {
        hipLaunchKernelGGL((mem_join_kernel<decltype(zero), decltype(lanes)::value, decltype(r)::value, (decltype(r)::value > 8)>), joins, dim3(256), 0, st, a, q->streams * x->query_heads, p.step);
        return d2c_check_launch("mem_join_kernel");
    };
    auto for_two = [&](bool yes, auto f) { return yes ? f(std::true_type{}) : f(std::false_type{}); };
    if (p.wide) {
        auto launch = [&](auto dp, auto r) {
            constexpr int DP = decltype(dp)::value, R = decltype(r)::value;
            const int rc = for_two(whole, [&](auto w) {
                return for_two(p.one, [&](auto one) {
                    hipLaunchKernelGGL((mem_attn_wide_kernel<DP, decltype(w)::value, R, decltype(one)::value>), grid, dim3(256), 0, st, a);
                    return d2c_check_launch("mem_attn_wide_kernel");
                });
            });
            if (rc || p.one) return rc;
            return join(bf16_t{}, std::integral_constant<int, DP <= 32 ? 8 : DP <= 64 ? 16 : 32>{}, r);
        };
        auto with_rows = [&](auto dp) { return p.rows == 16 ? launch(dp, std::integral_constant<int, 16>{}) : launch(dp, std::integral_constant<int, 32>{}); };
        if (q->D <= 32) return with_rows(std::integral_constant<int, 32>{});
        if (q->D <= 64) return with_rows(std::integral_constant<int, 64>{});
        if (q->D <= 96) return with_rows(std::integral_constant<int, 96>{});
        return with_rows(std::integral_constant<int, 128>{});
    }
    return for_rows(*q, a.group, [&](auto zero, auto lanes, auto r) {
        using T = decltype(zero);
        constexpr int LANES = decltype(lanes)::value, R = decltype(r)::value;
        const int rc = for_two(whole, [&](auto w) {
            return for_two(p.one, [&](auto one) {
                hipLaunchKernelGGL((mem_attn_kernel<T, LANES, R, decltype(w)::value, decltype(one)::value>), grid, dim3(256), 0, st, a);
                return d2c_check_launch("mem_attn_kernel");
            });
        });
        if (rc || p.one) return rc;
        return join(zero, std::integral_constant<int, LANES * 16 / (int)sizeof(T) / 4>{}, r);      // (lanes of four columns)
    });
}

// Streams whose ranks have room at once
int evict(const d2c_memory_desc *q, void *key, void *value, const int32_t *table, int32_t *lengths, const int32_t *seen, float *usage, int32_t *positions, int keep, int recent, void *ws,
          hipStream_t st)
{
    const EvictPlan p = evict_plan(*q, keep);
    EvictArgs a{};
    a.key = key; a.value = value; a.table = table; a.seen = seen; a.lengths = lengths; a.positions = positions; a.usage = usage;
    a.ranks = (uint32_t *)ws; a.holes = (int32_t *)((char *)ws + p.ranks_bytes); a.fillers = (int32_t *)((char *)ws + p.ranks_bytes + p.list_bytes);
    a.counts = (int32_t *)((char *)ws + p.ranks_bytes + 2 * p.list_bytes);
    for (int i = 0; i < 3; i++) { a.ks[i] = q->key_stride[i]; a.vs[i] = q->value_stride[i]; }
    a.table_stride = q->table_stride; a.slots_padded = p.slots_padded; a.page = make_fastdiv(q->page);
    a.N = q->streams; a.heads = q->heads; a.D = q->D; a.pages = q->pages; a.slots = q->per_stream * q->page; a.keep = keep; a.recent = recent; a.pairs = p.pairs;
    const int units = a.N * a.heads, vec = q->dtype == D2C_BF16 ? 8 : 4;
    hipLaunchKernelGGL(mem_rank_kernel, dim3(units), dim3(kEvictThreads), 0, st, a);
    if (int rc = d2c_check_launch("mem_rank_kernel")) return rc;
    const int blocks = (int)std::max(std::min((a.pairs + kMovePairs - 1L) / kMovePairs, (1L << 22) / units), 1L);
    const FastDiv pieces = make_fastdiv((a.D + vec - 1) / vec);
    if (q->dtype == D2C_BF16) hipLaunchKernelGGL(mem_move_kernel<bf16_t>, dim3((unsigned)blocks * units), dim3(256), 0, st, a, blocks, pieces);
    else hipLaunchKernelGGL(mem_move_kernel<float>, dim3((unsigned)blocks * units), dim3(256), 0, st, a, blocks, pieces);
    return d2c_check_launch("mem_move_kernel");
}

}  // namespace

extern "C" int d2c_memory_append(const d2c_memory_desc *q, void *key, void *value, const int32_t *table, int32_t *lengths, int32_t *seen,
                                 float *usage, int32_t *positions, const void *new_key, const void *new_value, const int64_t new_key_stride[2],
                                 const int64_t new_value_stride[2], const int32_t *starts, int64_t tokens, void *stream)
{
    if (int rc = check(q)) return rc;
    if (tokens < 0 || tokens >= (1L << 26) || (!starts && tokens != q->streams)) { d2c_set_error("memory_append: %ld tokens for %d streams", (long)tokens, q->streams); return D2C_ERR_SHAPE; }
    if (q->streams == 0) return D2C_OK;
    if (!lengths || !seen || (q->per_stream > 0 && !table) || (q->pages > 0 && (!key || !value || !usage || !positions)) || (tokens > 0 && (!new_key || !new_value)) ||
        !new_key_stride || !new_value_stride) {
        d2c_set_error("null tensor pointer");
        return D2C_ERR_SHAPE;
    }
    AppendArgs a{};
    a.nk = new_key; a.nv = new_value; a.key = key; a.value = value; a.table = table; a.starts = starts; a.lengths = lengths; a.seen = seen;
    a.positions = positions; a.usage = usage;
    for (int i = 0; i < 2; i++) { a.nks[i] = new_key_stride[i]; a.nvs[i] = new_value_stride[i]; }
    for (int i = 0; i < 3; i++) { a.ks[i] = q->key_stride[i]; a.vs[i] = q->value_stride[i]; }
    a.table_stride = q->table_stride; a.tokens = tokens; a.page = make_fastdiv(q->page);
    a.N = q->streams; a.heads = q->heads; a.D = q->D; a.pages = q->pages; a.slots = q->per_stream * q->page;
    hipStream_t st = (hipStream_t)stream;
    const bool half = q->dtype == D2C_BF16;
    if (!starts) {
        if (half) hipLaunchKernelGGL(mem_append_one_kernel<bf16_t>, dim3(a.N), dim3(256), 0, st, a);
        else hipLaunchKernelGGL(mem_append_one_kernel<float>, dim3(a.N), dim3(256), 0, st, a);
        return d2c_check_launch("mem_append_one_kernel");
    }
    if (tokens > 0) {
        const dim3 blocks((unsigned)((tokens + kAppendTokens - 1) / kAppendTokens));
        const FastDiv pieces = make_fastdiv((a.D * (half ? 2 : 4) + 15) / 16);
        if (half) hipLaunchKernelGGL(mem_append_kernel<bf16_t>, blocks, dim3(256), 0, st, a, pieces);
        else hipLaunchKernelGGL(mem_append_kernel<float>, blocks, dim3(256), 0, st, a, pieces);
        if (int rc = d2c_check_launch("mem_append_kernel")) return rc;
    }
    hipLaunchKernelGGL(mem_count_kernel, dim3((a.N + 255) / 256), dim3(256), 0, st, a);
    return d2c_check_launch("mem_count_kernel");
}

extern "C" size_t d2c_memory_attention_workspace_bytes(const d2c_memory_desc *q, const d2c_memory_query_desc *x, int32_t track)
{
    if (check(q, x) != D2C_OK || q->streams == 0) return 0;
    const int at_once = attention_streams(*q, *x, track != 0), last = (q->streams - 1) % at_once + 1;
    const size_t bytes = mem_plan(with_streams(*q, at_once), *x, track != 0).bytes;
    // (a smaller last part may take two launches where the others take one)
    return last == at_once ? bytes : std::max(bytes, mem_plan(with_streams(*q, last), *x, track != 0).bytes);
}

extern "C" int d2c_memory_attention(const d2c_memory_desc *q, const d2c_memory_query_desc *x, const void *query, const void *key,
                                    const void *value, const int32_t *table, const int32_t *lengths, float *usage, void *out, void *ws,
                                    size_t ws_bytes, void *stream)
{
    if (int rc = check(q, x)) return rc;
    if (q->streams == 0) return D2C_OK;
    const long slots = (long)q->per_stream * q->page;
    if (!query || !out || !lengths || (slots > 0 && !table) || (q->pages > 0 && (!key || !value))) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    const int at_once = attention_streams(*q, *x, usage != nullptr);
    if (at_once < q->streams)      // (before the first part runs)
        if (int rc = need(ws, ws_bytes, d2c_memory_attention_workspace_bytes(q, x, usage != nullptr))) return rc;
    const size_t size = d2c_elem_size(q->dtype);
    return for_streams(*q, at_once, [&](int n, const d2c_memory_desc &part) {
        return attend(&part, x, (const char *)query + n * x->query_stride[0] * size, key, value, table + n * q->table_stride, lengths + n, usage,
                      (char *)out + (size_t)n * x->query_heads * q->D * size, ws, ws_bytes, (hipStream_t)stream);
    });
}

extern "C" size_t d2c_memory_evict_workspace_bytes(const d2c_memory_desc *q, int32_t keep)
{
    if (check(q) != D2C_OK || keep <= 0) return 0;
    return evict_plan(with_streams(*q, evict_streams(*q, keep)), keep).bytes;
}

extern "C" int d2c_memory_evict(const d2c_memory_desc *q, void *key, void *value, const int32_t *table, int32_t *lengths, const int32_t *seen,
                                float *usage, int32_t *positions, int32_t keep, int32_t recent, void *ws, size_t ws_bytes, void *stream)
{
    if (int rc = check(q)) return rc;
    if (keep <= 0 || recent < 0 || recent > keep) { d2c_set_error("memory_evict: keep %d must be positive, recent %d in 0 .. keep", keep, recent); return D2C_ERR_SHAPE; }
    if (evict_plan(*q, keep).pairs == 0) return D2C_OK;
    if (!table || !lengths || !seen || (q->pages > 0 && (!key || !value || !usage || !positions))) { d2c_set_error("null tensor pointer"); return D2C_ERR_SHAPE; }
    if (int rc = need(ws, ws_bytes, d2c_memory_evict_workspace_bytes(q, keep))) return rc;
    return for_streams(*q, evict_streams(*q, keep), [&](int n, const d2c_memory_desc &part) {
        return evict(&part, key, value, table + n * q->table_stride, lengths + n, seen + n, usage, positions, keep, recent, ws, (hipStream_t)stream);
    });
}
