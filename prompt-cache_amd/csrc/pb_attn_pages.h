// What the kernels behind pcb_attn_pages share: how a call is cut, tiles, results.
#pragma once
#include "pb_pages.h"

#ifdef __HIPCC__
namespace pcb {

constexpr float LOG2E = 1.44269504088896f;
constexpr float NEG = -__builtin_inff();

constexpr int MANY_COLS = 128;
constexpr int MAX_GROUPS = 512;        // workgroups that share out the steps: two a CU
constexpr int SHARED_TILES = 512;      // tiles whose work is shared out evenly; more are enough units by themselves
constexpr int UNIT_STEPS = 8;          // what a unit costs beside its steps (queries, the first loads, the end), in steps
constexpr int MIN_SHARE = 8;           // the least that a workgroup takes, steps and units' costs together

struct Plan {
    int ps, per;                       // log2 of the page size; query heads of a key head
    uint32_t magic;                    // 2^32 / per, rounded up (per > 1)
    int cols, cblocks;                 // columns of a block, and the blocks of a full tile
    int groups;                        // few columns: workgroups that the steps are shared out to; 0: a workgroup takes all keys of its unit
    int runs, run;                     // many columns (cols = 128): key runs of a unit and their steps
    int halves;                        // .. and whether a workgroup is eight waves, two for each of its columns
};
// what `part` holds.  Few columns: the sums of the tiles' costs (int32 [n_tiles + 1]) and a workgroup's share, then for two results of each workgroup [cols][dim] and [cols][2];
// many columns: [dim] of each run of each (flat row, head), then all their pairs
__host__ __device__ inline int64_t head_floats(int n_tiles) { return ((int64_t)n_tiles + 2 + 3) / 4 * 4; }

// A unit of `steps` steps has place u0 among all costs, and shares of `share` cut through them: one that ends at place x of the unit ends it at this step, after a whole round of the four
// waves (or with the unit; ends inside a round: 20 rows of 32 heads over 2 000 keys 16.8 -> 21.1 us, 64 tokens over 8 192 the same)
__device__ __forceinline__ int step_at(int x, int steps) { return x >= steps + UNIT_STEPS ? steps : min(max((x - UNIT_STEPS + 2) / 4 * 4, 0), steps); }
// .. and the shares that have steps of it: the first that ends behind step 0, the last that starts in front of the end
__device__ __forceinline__ int first_share(int u0, int steps, int share) { return (int)((uint32_t)(u0 + UNIT_STEPS + min(1, steps - 1)) / (uint32_t)share); }
__device__ __forceinline__ int last_share(int u0, int steps, int share) { return (int)((uint32_t)(u0 + UNIT_STEPS + min((steps + 3) / 4 * 4 - 3, steps - 1)) / (uint32_t)share); }

// x / per for x per < 2^32
__device__ __forceinline__ int row_of(const Plan& pl, int x) { return pl.per == 1 ? x : (int)__umulhi((uint32_t)x, pl.magic); }

// e^x of differences of running maxima, in the units that the type keeps them in
template <typename E>
__device__ __forceinline__ float pow_of(float x) { return __builtin_amdgcn_exp2f(sizeof(E) == 4 ? x * LOG2E : x); }

// Maxima beyond this are far: fp32 numbers there are 2^-3 or more apart, in the end further than e.  Then a weight's exponent is taken from the same rounded number that the maximum was
// (one fma of the sum of products, less M: the largest is 0 exactly), not from the exact product less another rounding: half a step of M would make the largest weight more than a
// half holds, or 0.  Up to it the exponent is off by 2^-3 at most, of numerator and denominator alike.
constexpr float FAR = 1048576.0f;
// .. such a sum of products, in units of 1: what it is above M, less ln vs, which the exponent gets again
__device__ __forceinline__ float above(float s, float f, float lv, float M) { return __builtin_fmaf(s, f, lv) - M - lv; }

// What a sum of products of a query and a key stands for.  Above 0 and finite whatever the two are (a row of zeros over the smallest scale would give 0, and -infinity, a key that is
// not seen, times 0 is no number); sums that this changes are 0 or too small to count, or beyond all numbers
__device__ __forceinline__ float score_unit(float qs, float ks) { return __builtin_fminf(__builtin_fmaxf(qs * ks, 1.17549435e-38f), 3.40282347e38f); }

// e^(x - M) of an fp32 score x = s f: 2^p e^(d - p ln 2) with p = d log2 e as it was rounded, so that the error does not grow with |d| by more than 2^-28 of it.  What is no number
// comes out as one (or_not)
__device__ __forceinline__ float exp_of_score(float s, float f, float M) {
    const float d = __builtin_fmaxf(__builtin_fmaf(s, f, -M), -200.0f), p = d * 1.44269502e+00f, q = __builtin_amdgcn_exp2f(p);
    return __builtin_fmaf(q, __builtin_fmaf(p, -6.93147182e-01f, d), q);
}
// A sum of scores is no number if one of them is none (or some are infinite and some -infinity, whose exponentials have no sum either): a step's sum of exponentials then
__device__ __forceinline__ float or_not(float sum, float scores) { return scores == scores ? sum : scores; }
// a weight as two halves
__device__ __forceinline__ void two_halves(float w, _Float16& hi, _Float16& lo) {
    hi = (_Float16)w;
    lo = (_Float16)__builtin_fmaf((float)hi, -1.0f, w);
}

// the quotient of a column: its sums under the maximum m, and the sink.  No score above -infinity: 0, but scores that are no numbers stay so
template <typename E>
__device__ __forceinline__ float finished(const pcb_attn_pages_args& a, int h, float m, float den, float num) {
    if (m == NEG) return den * 0.0f;
    if (a.sink) den += __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (a.sink[h] - m) * LOG2E : a.sink[h] * LOG2E - m);
    return num * (1.0f / 16384.0f) / den;
}

// a tile as the kernels take it: no rows where it is of no sequence or reaches out of the rows; and the steps of 64 keys [s0, s1) that some of its rows see
struct Tile {
    int seq, pos, rows, row0, kv, s0, s1;
};
// the tile with the steps that its rows first .. last see
__device__ __forceinline__ Tile rows_of(const pcb_attn_pages_args& a, Tile x, int first, int last) {
    const int end = (int)min((int64_t)x.kv, (int64_t)x.pos + last + 1);
    int begin = a.window > 0 ? x.pos + first - a.window + 1 : 0;
    begin = begin < 0 ? 0 : begin;
    x.s0 = begin >> 6, x.s1 = end > begin ? (end + 63) >> 6 : x.s0;
    return x;
}
__device__ __forceinline__ Tile tile_of(const pcb_attn_pages_args& a, int t, int ps) {
    const int4 r = reinterpret_cast<const int4*>(a.tiles)[t];
    Tile x;
    x.seq = r.x, x.pos = r.y, x.rows = r.z < a.tile_rows ? r.z : a.tile_rows, x.row0 = r.w;
    x.kv = 0, x.s0 = 0, x.s1 = 0;
    if (r.x < 0 || r.x >= a.n_seqs || r.y < 0 || r.w < 0 || x.rows <= 0 || r.y > 0x7fffffff - x.rows || (int64_t)r.w + x.rows > a.n_rows) {
        x.rows = 0;
        return x;
    }
    x.kv = (int)min((int64_t)a.kv_len[r.x], (int64_t)a.max_pages << ps);
    return rows_of(a, x, 0, x.rows - 1);
}

}  // namespace pcb

// tiles of many columns (pb_attn_pages_prompt.hip)
int pcb_attn_pages_prompt(const pcb_attn_pages_args& a, const pcb::Plan& pl, hipStream_t stream);
#endif
