// pcb_attn_pages: causal softmax attention over keys and values held in 8 bits in pages, a power-of-two scale for each page and key head.  Here for blocks of 16 or 32 columns.
//
// Queries and heads of one key head are COLUMNS of a tile: column = row * (H / Hkv) + head, so a key or value is read and made a number once for all heads that
// share it.  S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16: codes of both kinds are halves exactly, a query row divided by the power of two
// of its largest element is (bf16) or is as the sum of two halves (fp32, 22 bits), and softmax weights are 11 bits (fp32: 22).  All sums are fp32.
//
// A bf16 row's weights enter the second product as one half.  The attention of this library whose operands are bf16 has them as a pair, 17 bits, for one bf16 has 8, no more than the
// result; a half's 11 move a result by 1.0 to 3.0e-4 of its norm, where its own rounding is 1.6e-3, and its distance from 64 bits by nothing that shows: 64 tokens over up to 7 786 keys
// 1.587e-3, with two halves and in 32 bits 1.586e-3; 3 989 prompt rows 1.574e-3 all three.  Two halves cost the prompts 491 -> 629 us, 27 rows over 8 274 keys 29.1 -> 32.8, single
// tokens 47.0 -> 47.2.  fp32 rows, two halves of queries and weights: off by 4.6e-7 (prompts) and 4.9e-7 (two tokens) of the norm, products and sums of 24 bits by 8.6e-7 and 5.5e-7.
//
// Scales never touch an operand: a page's key scale multiplies its scores.  The second product takes w = e^(s - M) vscale, M the running maximum of s + ln vscale
// over the keys a column has seen (so w <= 1 whatever the scales are, held as w 2^14 to keep halves normal down to 2^-28); the denominator sums e^(s - M) itself.
//
// A step walks 64 keys.  Lane group g (16 lanes) owns the sixteen keys 16 g .. 16 g + 15 of the step, in every role: which key a row of the first product's operand is may
// be chosen freely, so row 4 g + r of its block b is key 16 g + 4 b + r, and the lane's scores are then, in order, the keys of its operand of the second product, sixteen
// neighbouring codes of a value column, one 16-byte load.  Pages have at least 16 tokens: a lane needs one page number and one pair of scales a step.
//
// Bound by the codes' bytes, which are read once, and before them by a chain of loads that each need the one before (tile, length, page number, keys: ~6 us of a launch).  Measured
// (the launch alone, over caches that change from one to the next; bf16, 4 heads a key head of 128): 64 single tokens over up to 7 786 keys, 189 MB, 47.8 us = 4.0 TB/s; one over
// 131 072, 268 MB, 54.3 us = 4.9 TB/s, 7.6 more its merge; 27 rows over 8 274 keys of 32 heads, 68 MB, 28.3 us and 5.9: a wave has two steps of its own there.  (The same cache again and
// again, which the last-level cache holds in part: 37.7, 44.4 and 25.5.)  A copy reaches 4.9 TB/s, a reading stream ~5.9.  fp32 rows: the batch of tokens 49.5 us, the long one 63.7
// with its merge, the 27 rows 58.
#include "pb_attn_pages.h"

namespace {
using namespace pcb;

__device__ __forceinline__ float max4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Sixteen neighbouring elements of a query row, as they are in memory
template <typename E>
struct Query {
    u32x4 w[sizeof(E)];
    __device__ __forceinline__ float at(int e) const {
        if constexpr (sizeof(E) == 2)
            return __uint_as_float(e & 1 ? w[e >> 3][(e & 7) >> 1] & 0xffff0000u : w[e >> 3][(e & 7) >> 1] << 16);
        else
            return __uint_as_float(w[e >> 2][e & 3]);
    }
};
// .. as halves (PARTS = 2: sums of two) at `to` (null: only looked at), the second ones `parts` behind.  THREADS neighbouring lanes, all of them here, hold a row.  -> the power of two that the row was divided by: its largest
// element becomes 2^14 .. 2^15, and what is 2^-28 of that is still a normal half
template <typename E, int PARTS, int THREADS>
__device__ __forceinline__ float as_halves(const Query<E>& q, _Float16* to, int parts) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, __builtin_fabsf(q.at(e)) < __builtin_inff() ? __builtin_fabsf(q.at(e)) : 0.0f);
#pragma unroll
    for (int o = 1; o < THREADS; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    int e2 = (int)(__float_as_uint(m) >> 23) - 127 - 14;
    e2 = e2 < -110 ? -110 : e2;
    const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        h8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = q.at(8 * k + e) * inv;
            hi[e] = (_Float16)y;
            if constexpr (PARTS == 2) lo[e] = __builtin_fabsf(y) < __builtin_inff() ? (_Float16)(y - (float)hi[e]) : (_Float16)0.0f;
        }
        if (!to) continue;
        *reinterpret_cast<h8*>(to + 8 * k) = hi;
        if constexpr (PARTS == 2) *reinterpret_cast<h8*>(to + parts + 8 * k) = lo;
    }
    return __uint_as_float((uint32_t)(127 + e2) << 23);
}

// Sixteen scores of a lane (in units of 1 / f; -infinity: not seen) as weights of the second product: w = e^(s - M) vs 2^14 with M the running maximum of s + ln vs over the
// column's keys; l += the lane's part of sum e^(s - M); alpha: what earlier results are multiplied with.
template <typename E, int PARTS>
__device__ __forceinline__ void weights(f4 (&acc)[4], float f, float vs, float& M, float& l, float& alpha, h8 (&wf)[PARTS][2]) {
    float top = NEG;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, acc[i >> 2][i & 3]);
    const float lvs = exp_of(vs), lv = PARTS == 2 ? lvs * 0.693147181f : lvs;
    top = max4(__builtin_fmaf(top, f, lv));                           // (f > 0)
    const float M_new = fmaxf(M, top);
    float M_use = M_new == NEG ? 0.0f : M_new;
    alpha = pow_of<E>(M - M_use);
    M = M_new;
    if (__builtin_expect(__builtin_fabsf(M_use) > FAR, 0)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i >> 2][i & 3] = above(acc[i >> 2][i & 3], f, lv, M_use);
        f = 1.0f, M_use = 0.0f;
    }
    float sum = 0.0f;
    if constexpr (PARTS == 1) {
        // vs and 2^14 inside the exponent, out of the sum again: all powers of two
        const float off = lvs + 14.0f - M_use;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i >> 2][i & 3], f, off));
            sum += w;
            wf[0][i >> 3][i & 7] = (_Float16)w;
        }
        sum *= inv_pow2(vs) * (1.0f / 16384.0f);
    } else {
        const float up = vs * 16384.0f;
        float scores = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = exp_of_score(acc[i >> 2][i & 3], f, M_use);
            scores += acc[i >> 2][i & 3];
            sum += e;
            _Float16 hi, lo;
            two_halves(e * up, hi, lo);
            wf[0][i >> 3][i & 7] = hi, wf[1][i >> 3][i & 7] = lo;
        }
        sum = or_not(sum, scores);
    }
    l = l * alpha + sum;
}

// Numbers that one workgroup leaves for another one of the same launch: written through and read past the caches, which differ between XCDs.
__device__ __forceinline__ void hand_on(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 handed(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

// one more result of a column: maximum, denominator, sums
template <typename E, int DB>
__device__ __forceinline__ void add_result(float& m, float& den, f4 (&v)[DB], float mi, float li, const f4 (&vi)[DB]) {
    const float mn = fmaxf(m, mi), mu = mn == NEG ? 0.0f : mn, x = pow_of<E>(m - mu), y = pow_of<E>(mi - mu);
    m = mn, den = den * x + li * y;
#pragma unroll
    for (int k = 0; k < DB; ++k) v[k] = v[k] * x + vi[k] * y;
}

// A unit is 16 NC columns of a tile and one key head.  The steps of all units, one after the other, are shared out evenly: a workgroup's share may begin inside a unit and
// end inside another one; what is not a whole unit goes to `part`.  So sequences of any lengths fill the chip alike, and no workgroup starts in vain.  A unit without steps
// counts as one: its rows get their zeros.
//
// Within a unit the waves take steps in turns.  Keys and values go from memory straight into operand registers: a step's values are under way during its softmax, the next
// step's keys as soon as this one's values have been multiplied, and the two take turns in the same registers; nothing crosses waves but the end.  (Both with registers of
// their own, a step ahead: no faster with two workgroups a CU, and the same with three or four, which their registers then only allow with spills, 1.1 to 1.6 x the time.)
template <typename E, int CODE, int DB, int NC>
__global__ __launch_bounds__(256, 2) void attn_pages_rows_kernel(pcb_attn_pages_args a, Plan pl) {
    constexpr bool F32 = sizeof(E) == 4;
    constexpr int NW = 4, NT = 256, PARTS = F32 ? 2 : 1, NB = 4 * DB, COLS = 16 * NC;   // NB: value column blocks of 16
    constexpr int TPC = DB == 1 ? 4 : DB == 2 ? 8 : 16, QLD = 64 * DB + 8;            // threads that bring a query row, and a row of halves
    static_assert(COLS * TPC <= NT && COLS * QLD * PARTS * 2 <= NW * 16 * (64 * DB + 4) * 4, "a pass, in the results' place");
    __shared__ __attribute__((aligned(16))) float Os[NW][16][64 * DB + 4];
    _Float16* const Qs = reinterpret_cast<_Float16*>(&Os[0][0][0]);  // (before there are results)
    __shared__ float Ms[NW][COLS], Ls[NW][COLS];
    __shared__ __attribute__((aligned(16))) int4 tiles_s[SHARED_TILES];
    __shared__ int starts[SHARED_TILES + 1], kv_s[SHARED_TILES], wsum[NW], last_s;
    __shared__ float unit_s[COLS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = pl.per, dim = a.dim, ps = pl.ps, P = 1 << ps;
    const int64_t plane = (int64_t)P * dim;
    // Heads of less than 64 DB elements: what lies behind reads a head's last sixteen again (numbers, times the queries' zeros) or a column block that nobody stores
    const int last_b = dim / 16 - 1;
    int at = 0, end = 1, share = 1;
    if (pl.groups) {
        const int tid = threadIdx.x, lane = tid & 63;
        int all = 0;
        auto cost_of = [&](int t) {
            if (t >= a.n_tiles) return 0;
            const Tile x = tile_of(a, t, ps);
            tiles_s[t] = int4{x.seq, x.pos, x.rows, x.row0}, kv_s[t] = x.kv;
            return (max(x.s1 - x.s0, 1) + UNIT_STEPS) * a.Hkv * ((x.rows * per + COLS - 1) / COLS);
        };
        if (a.n_tiles <= 64) {                                        // (every wave for itself: the same numbers)
            const int n = cost_of(lane), v = wave_scan(n);
            if (lane < a.n_tiles) starts[lane] = v - n;
            all = __builtin_amdgcn_readlane(v, 63);
        }
        for (int t0 = 0; a.n_tiles > 64 && t0 < a.n_tiles; t0 += NT) {
            const int n = cost_of(t0 + tid);
            int v = wave_scan(n);
            if (lane == 63) wsum[wave] = v;
            __syncthreads();
            int sum = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                if (w < wave) v += wsum[w];
                sum += wsum[w];
            }
            if (t0 + tid < a.n_tiles) starts[t0 + tid] = all + v - n;
            all += sum;
            __syncthreads();
        }
        all = __builtin_amdgcn_readfirstlane(all);
        share = (all + pl.groups - 1) / pl.groups;
        share = share < MIN_SHARE ? MIN_SHARE : share;
        if (tid == 0) starts[a.n_tiles] = all;
        __syncthreads();
        if (blockIdx.x == 0 && !a.counters) {                         // for the launch that merges
            int* head = reinterpret_cast<int*>(a.part);
            for (int t = tid; t <= a.n_tiles; t += NT) head[t] = starts[t];
            if (tid == 0) head[a.n_tiles + 1] = share;
        }
        at = blockIdx.x * share, end = min(at + share, all);
    }
    const int at0 = at;
    float* const part = a.part + head_floats(a.n_tiles);
    while (at < end) {
        int t, j, from, steps, n_steps, mine = 1, u0 = 0;    // unit j of tile t, whose place among all is u0; its steps from .. from + n_steps - 1
        Tile tl;
        if (pl.groups) {
            t = 0;
            for (int i = threadIdx.x & 63; t < a.n_tiles; i += 64, t += 64) {   // (every wave by itself; `at` is in one)
                const uint64_t here = __ballot(i < a.n_tiles && starts[i] <= at && at < starts[i + 1]);
                if (here) {
                    t += __builtin_ctzll(here);
                    break;
                }
            }
            const int4 rec = tiles_s[t];
            tl.seq = __builtin_amdgcn_readfirstlane(rec.x), tl.pos = __builtin_amdgcn_readfirstlane(rec.y), tl.rows = __builtin_amdgcn_readfirstlane(rec.z);
            tl.row0 = __builtin_amdgcn_readfirstlane(rec.w), tl.kv = __builtin_amdgcn_readfirstlane(kv_s[t]);
            tl = rows_of(a, tl, 0, tl.rows - 1);
            steps = max(tl.s1 - tl.s0, 1);
            const int off = at - __builtin_amdgcn_readfirstlane(starts[t]), cost = steps + UNIT_STEPS;
            j = (int)((uint32_t)off / (uint32_t)cost);
            const int p = off - j * cost;
            mine = min(cost - p, end - at);
            u0 = at - p;
            from = step_at(p, steps), n_steps = step_at(p + mine, steps) - from;
        } else {
            t = blockIdx.x, j = blockIdx.y;
            tl = tile_of(a, t, ps);
            from = 0, steps = n_steps = max(tl.s1 - tl.s0, 1);
            if (j / a.Hkv * COLS >= tl.rows * per) return;
        }
        const bool unit = n_steps == steps;
        const int slot = unit ? 0 : 2 * (int)blockIdx.x + (at == at0 ? 0 : 1);
        at += mine;
        if (n_steps == 0) continue;                                   // (the share ends in front of the unit's first steps, or begins behind its last ones)
        int tid = threadIdx.x;
        asm("" : "+v"(tid));                                          // (what hangs on it is computed anew for every unit: kept over the loop it takes the inner one's registers)
        const int lane = tid & 63, g = lane >> 4, c = lane & 15;
        const int cblock = j / a.Hkv, hk = j - cblock * a.Hkv, col0 = cblock * COLS, rows = tl.rows, kv = tl.kv;
        const int s0 = tl.s0 + from, s1 = min(s0 + n_steps, tl.s1);
        const int last_col = min(col0 + COLS, rows * per) - 1;
        // keys that all of the unit's columns see
        const int all_lo = a.window > 0 ? tl.pos + row_of(pl, last_col) - a.window + 1 : 0, all_hi = min(kv, tl.pos + row_of(pl, col0) + 1);
        int lo[NC], hi[NC];                                           // a column's keys [lo, hi)
        float qs[NC];
        h8 qf[NC][PARTS][2 * DB];
        const int32_t* table = a.table + (int64_t)tl.seq * a.ld_table;
        // pages and scales of sixteen of the wave's steps at once: lane 4 i + k those of its step i's keys 16 k ..
        int pages = -1;
        float kss = 1.0f, vss = 1.0f;
        auto look = [&](int s) {
            const int key = (s + (lane >> 2) * NW) * 64 + 16 * (lane & 3);
            pages = s + (lane >> 2) * NW < s1 && key < kv ? table[key >> ps] : -1;
            pages = pages >= 0 && pages < a.n_pages ? pages : -1;
            const int64_t ph = (int64_t)(pages < 0 ? 0 : pages) * a.Hkv + hk;
            kss = pages < 0 ? 1.0f : a.kscale[ph], vss = pages < 0 ? 1.0f : a.vscale[ph];
        };
        u32x4 kr[4][DB], vr[NB];
        auto fetch_k = [&](int s, int i) {
            const int page = __shfl(pages, 4 * i + (c >> 2), 64);     // of the sixteen keys that row c of the first product's operand is one of
            const int row = ((s * 64 + 16 * (c >> 2)) & (P - 1)) + (c & 3);
            const uint8_t* p = (const uint8_t*)a.kcodes + ((int64_t)(page < 0 ? 0 : page) * a.Hkv + hk) * plane + row * dim;
#pragma unroll
            for (int ch = 0; ch < DB; ++ch) {
                const uint8_t* q = p + 16 * min(4 * ch + g, last_b);
                asm("" : "+v"(q));                                    // (one address and steps that all lanes share, not sixteen sums kept over the loop)
#pragma unroll
                for (int b = 0; b < 4; ++b) kr[b][ch] = *reinterpret_cast<const u32x4*>(q + 4 * b * dim);
            }
        };
        auto fetch_v = [&](int s, int i) {
            const int page = __shfl(pages, 4 * i + g, 64);
            const uint8_t* p = (const uint8_t*)a.vcodes + ((int64_t)(page < 0 ? 0 : page) * a.Hkv + hk) * plane + ((s * 64 + 16 * g) & (P - 1)) + c * P;
            asm("" : "+v"(p));
#pragma unroll
            for (int b = 0; b < NB; ++b) vr[b] = *reinterpret_cast<const u32x4*>(p + 16 * min(b, last_b) * P);
        };
        // The queries are asked for first, sixteen elements a thread: loads arrive in order, and they are made halves while the first keys are under way, once for all waves.  (Every
        // wave its own operands instead: 500 instructions more for each 16 columns before the first product, 27 rows of 32 heads over 8 274 keys 29.6 -> 33.6 us.)
        const int qc = tid / TPC, qk = tid % TPC;
        Query<E> raw;
#pragma unroll
        for (int k = 0; k < (int)sizeof(E); ++k) raw.w[k] = u32x4{0, 0, 0, 0};   // (behind a row's end, and where the column is nobody's)
        if (col0 + qc <= last_col && qk <= last_b && qc < COLS) {
            const int col = col0 + qc, qr = row_of(pl, col), h = hk * per + col - qr * per;
            const E* q = (const E*)a.q + ((int64_t)tl.row0 + qr) * a.ldq + (int64_t)h * a.q_head_stride + 16 * qk;
#pragma unroll
            for (int k = 0; k < (int)sizeof(E); ++k) raw.w[k] = *reinterpret_cast<const u32x4*>(q + k * (16 / sizeof(E)));
        }
        int s = s0 + wave, i = 0;
        if (s < s1) {
            look(s);
            fetch_k(s, 0);
        }
        {
            const float unit2 = as_halves<E, PARTS, TPC>(raw, qc < COLS && qk < 4 * DB ? Qs + qc * QLD + 16 * qk : nullptr, COLS * QLD);
            if (qc < COLS && qk == 0) unit_s[qc] = F32 ? unit2 * a.scale : unit2 * (a.scale * LOG2E);   // bf16: scores in units of ln 2
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int col = col0 + 16 * n + c;
            const bool live = col < rows * per;
            const int pos = live ? tl.pos + row_of(pl, col) : -1;
            lo[n] = a.window > 0 ? pos - a.window + 1 : 0, hi[n] = min(kv, pos + 1);
            qs[n] = unit_s[16 * n + c];
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int k = 0; k < 2 * DB; ++k) qf[n][p][k] = *reinterpret_cast<const h8*>(Qs + (p * COLS + 16 * n + c) * QLD + 64 * (k >> 1) + 16 * g + 8 * (k & 1));
        }
        float M[NC], l[NC];
        f4 o[NC][NB];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            M[n] = NEG, l[n] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) o[n][b] = f4{0.f, 0.f, 0.f, 0.f};
        }
        for (; s < s1; s += NW) {
            f4 acc[NC][4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
#pragma unroll
                for (int n = 0; n < NC; ++n) acc[n][b] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ch = 0; ch < DB; ++ch) {
                    const h8 k0 = half8<CODE>(u32x2{kr[b][ch][0], kr[b][ch][1]}), k1 = half8<CODE>(u32x2{kr[b][ch][2], kr[b][ch][3]});
#pragma unroll
                    for (int n = 0; n < NC; ++n)
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) {
                            acc[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[n][p][2 * ch], acc[n][b], 0, 0, 0);
                            acc[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[n][p][2 * ch + 1], acc[n][b], 0, 0, 0);
                        }
                }
            }
            const int key0 = s * 64 + 16 * g;
            const int page = __shfl(pages, 4 * i + g, 64);
            const float ks = __shfl(kss, 4 * i + g, 64), vs = __shfl(vss, 4 * i + g, 64);
            const bool more = s + NW < s1;
            const int i_next = (i + 1) & 15;
            __builtin_amdgcn_sched_barrier(0);                        // (the phases' registers do not overlap; loads drawn ahead into the one before would make them)
            fetch_v(s, i);
            // a step that all columns see whole needs no comparisons
            const bool seen = s * 64 + 64 <= all_hi && s * 64 >= all_lo && __all(page >= 0);
            h8 wf[NC][PARTS][2];
            float alpha[NC];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (!seen) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = key0 + e;
                        if (!(page >= 0 && key >= lo[n] && key < hi[n])) acc[n][e >> 2][e & 3] = NEG;
                    }
                }
                weights<E, PARTS>(acc[n], score_unit(qs[n], ks), vs, M[n], l[n], alpha[n], wf[n]);
            }
            __builtin_amdgcn_sched_barrier(0);
            // values: codes behind the last written key are whatever the memory held, and no number times 0 is 0 for all of them
            if (!seen) {
                const int have = page < 0 ? 0 : kv - key0;
                uint32_t keep[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = have - 4 * e;
                    keep[e] = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : 0xffffffffu >> (32 - 8 * k);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) vr[b][e] &= keep[e];
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const h8 v0 = half8<CODE>(u32x2{vr[b][0], vr[b][1]}), v1 = half8<CODE>(u32x2{vr[b][2], vr[b][3]});
#pragma unroll
                for (int n = 0; n < NC; ++n) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[n][b][r] *= alpha[n];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, wf[n][p][0], o[n][b], 0, 0, 0);
                        o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, wf[n][p][1], o[n][b], 0, 0, 0);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (more) {
                if (i_next == 0) look(s + NW);
                fetch_k(s + NW, i_next);
            }
            i = i_next;
        }
        // the waves' results under one maximum, sixteen columns after sixteen: sixteen threads a column, four neighbouring elements each
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            l[n] = sum4(l[n]);
            if (g == 0) Ms[wave][16 * n + c] = M[n], Ls[wave][16 * n + c] = l[n];
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            __syncthreads();
            float top = NEG;
#pragma unroll
            for (int w = 0; w < NW; ++w) top = fmaxf(top, Ms[w][16 * n + c]);
            const float back = pow_of<E>(M[n] - (top == NEG ? 0.0f : top));
#pragma unroll
            for (int b = 0; b < NB; ++b) *reinterpret_cast<f4*>(&Os[wave][c][16 * b + 4 * g]) = o[n][b] * back;
            __syncthreads();
            const int cc = tid >> 4, col = col0 + 16 * n + cc;
            if (col >= rows * per) continue;
            float m = NEG, den = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) m = fmaxf(m, Ms[w][16 * n + cc]);
#pragma unroll
            for (int w = 0; w < NW; ++w) den += Ls[w][16 * n + cc] * pow_of<E>(Ms[w][16 * n + cc] - (m == NEG ? 0.0f : m));
            const int qr = row_of(pl, col), h = hk * per + col - qr * per;
            float* pp = part + (int64_t)slot * COLS * (dim + 2);
            E* op = (E*)a.out + ((int64_t)tl.row0 + qr) * a.ldo + (int64_t)h * a.out_head_stride;
            const float f = unit ? finished<E>(a, h, m, den, 16384.0f) * (1.0f / 16384.0f) : 1.0f;
            if (!unit && (tid & 15) == 0) hand_on(pp + COLS * dim + 2 * (16 * n + cc), m, den);
            for (int d = 4 * (tid & 15); d < dim; d += 64) {
                f4 v = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const f4*>(&Os[w][cc][d]);
                if (unit)
                    store4(op + d, v[0] * f, v[1] * f, v[2] * f, v[3] * f);
                else
                    hand_on(pp + (16 * n + cc) * dim + d, v[0], v[1]), hand_on(pp + (16 * n + cc) * dim + d + 2, v[2], v[3]);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");              // (every wave's results have left it before one of them answers for all)
        __syncthreads();
        if (unit || !a.counters) continue;
        // the workgroups that share the unit: g0 .. g0 + parts - 1, the first one's result its second where it had another unit's before
        const int g0 = first_share(u0, steps, share), parts = last_share(u0, steps, share) - g0 + 1, second = u0 > g0 * share;
        // The last of the unit's workgroups merges: its fellows' results were past the caches before they were counted.
        if (tid == 0) {
            last_s = __hip_atomic_fetch_add(&a.counters[g0], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
            if (last_s) __hip_atomic_store(&a.counters[g0], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_s) continue;
        // Sixteen threads a column, and more sets of sixteen where there are fewer columns: each adds up every so many of the results under a running maximum, then the sets' sums are
        // put together.  (A wave a column instead, its maximum first: 32 columns of 15 results 18 us longer than the second launch that this saves.)
        const int64_t result = (int64_t)COLS * (dim + 2);
        auto place = [&](int i) { return part + (2 * (int64_t)(g0 + i) + (i == 0 ? second : 0)) * result; };
        float* sums = &Os[0][0][0];                                   // [16][64 DB + 4]
        for (int n = 0; n < NC; ++n) {
            const int n_live = min(16, rows * per - col0 - 16 * n);
            if (n_live <= 0) break;
            const int wide = n_live == 1 ? 1 : 1 << (32 - __builtin_clz(n_live - 1)), grp = tid >> 4, q = tid & 15;   // (a power of two of columns)
            const int cc = 16 * n + (grp & (wide - 1)), set = grp / wide, sets = 16 / wide;
            float m = NEG, den = 0.0f;
            f4 v[DB];
#pragma unroll
            for (int k = 0; k < DB; ++k) v[k] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int i = set; i < parts; i += sets) {
                const float* p = place(i);
                const float2 x = handed(p + COLS * dim + 2 * cc);
                f4 w[DB];
#pragma unroll
                for (int k = 0; k < DB; ++k) {
                    const int d = min(4 * q + 64 * k, dim - 4);
                    const float2 y = handed(p + cc * dim + d), z = handed(p + cc * dim + d + 2);
                    w[k] = f4{y.x, y.y, z.x, z.y};
                }
                add_result<E, DB>(m, den, v, x.x, x.y, w);
            }
            float* mine_s = sums + grp * (64 * DB + 4);
            if (sets > 1) {
                __syncthreads();                                      // (`sums` of the columns before have been read)
#pragma unroll
                for (int k = 0; k < DB; ++k) *reinterpret_cast<f4*>(mine_s + 4 * q + 64 * k) = v[k];
                if (q == 0) mine_s[64 * DB] = m, mine_s[64 * DB + 1] = den;
                __syncthreads();
                for (int k = 1; k < sets && set == 0; ++k) {
                    const float* o = sums + (grp + k * wide) * (64 * DB + 4);
                    f4 w[DB];
#pragma unroll
                    for (int e = 0; e < DB; ++e) w[e] = *reinterpret_cast<const f4*>(o + 4 * q + 64 * e);
                    add_result<E, DB>(m, den, v, o[64 * DB], o[64 * DB + 1], w);
                }
            }
            if (set > 0 || cc - 16 * n >= n_live) continue;
            const int col = col0 + cc, qr = row_of(pl, col), h = hk * per + col - qr * per;
            const float f = finished<E>(a, h, m, den, 16384.0f) * (1.0f / 16384.0f);
            E* op = (E*)a.out + ((int64_t)tl.row0 + qr) * a.ldo + (int64_t)h * a.out_head_stride;
#pragma unroll
            for (int k = 0; k < DB; ++k)
                if (4 * q + 64 * k < dim) store4(op + 4 * q + 64 * k, v[k][0] * f, v[k][1] * f, v[k][2] * f, v[k][3] * f);
        }
        __syncthreads();
    }
}

// The results of the workgroups that shared a unit, put together in a launch of their own: sixteen threads a (row, head), or `sets` times as many where there are many results, each
// adds up every so many of them under a running maximum.
template <typename E, int DB>
__global__ __launch_bounds__(256) void attn_pages_merge_kernel(pcb_attn_pages_args a, Plan pl, int sets) {
    __shared__ __attribute__((aligned(16))) float sums[16][64 * DB + 4];
    const int dim = a.dim, per = pl.per, grp = threadIdx.x >> 4, q = threadIdx.x & 15, wide = 16 / sets, set = grp / wide;
    const int blocks = (a.tile_rows * a.H + wide - 1) / wide, t = blockIdx.x / blocks, item = (blockIdx.x - t * blocks) * wide + (grp & (wide - 1)), r = item / a.H, h = item - r * a.H;
    const Tile tl = tile_of(a, t, pl.ps);
    const int hk = row_of(pl, h), col = r * per + h - hk * per, cblock = col / pl.cols, cc = col - cblock * pl.cols;
    // the column's first result (sums, maximum and denominator), its second, and how far it is from there to the next
    const float *sum0 = a.part, *sum1 = a.part, *max0 = a.part, *max1 = a.part;
    int64_t sum_step = 0, max_step = 0;
    int n = 0;
    if (r < tl.rows && pl.cols == MANY_COLS) {
        const Tile bl = rows_of(a, tl, row_of(pl, cblock * MANY_COLS), row_of(pl, min(cblock * MANY_COLS + MANY_COLS, tl.rows * per) - 1));
        n = min((bl.s1 - bl.s0 + pl.run - 1) / pl.run, pl.runs);
        const int64_t i = (((int64_t)tl.row0 + r) * a.H + h) * pl.runs;
        sum0 = a.part + i * dim, max0 = a.part + (int64_t)a.n_rows * a.H * pl.runs * dim + 2 * i;
        sum1 = sum0 + dim, max1 = max0 + 2, sum_step = dim, max_step = 2;
    } else if (r < tl.rows) {
        const int* head = reinterpret_cast<const int*>(a.part);
        const float* part = a.part + head_floats(a.n_tiles);
        const int64_t result = (int64_t)pl.cols * (dim + 2);
        const int share = head[a.n_tiles + 1];
        const int steps = max(tl.s1 - tl.s0, 1), u0 = head[t] + (steps + UNIT_STEPS) * (cblock * a.Hkv + hk);   // the unit's place among all
        const int g0 = first_share(u0, steps, share);
        n = last_share(u0, steps, share) - g0 + 1;
        const float *first = part + (2 * (int64_t)g0 + (u0 > g0 * share ? 1 : 0)) * result, *second = part + 2 * ((int64_t)g0 + 1) * result;
        sum0 = first + cc * dim, max0 = first + pl.cols * dim + 2 * cc, sum1 = second + cc * dim, max1 = second + pl.cols * dim + 2 * cc, sum_step = max_step = 2 * result;
    }
    n = n <= 1 ? 0 : n;                                               // (one workgroup had it all)
    float m = NEG, den = 0.0f;
    f4 v[DB];
#pragma unroll
    for (int k = 0; k < DB; ++k) v[k] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = set; i < n; i += sets) {
        const float *p = i == 0 ? sum0 : sum1 + sum_step * (i - 1), *mp = i == 0 ? max0 : max1 + max_step * (i - 1);
        const float2 x = *reinterpret_cast<const float2*>(mp);
        f4 w[DB];
#pragma unroll
        for (int k = 0; k < DB; ++k) w[k] = *reinterpret_cast<const f4*>(p + min(4 * q + 64 * k, dim - 4));
        add_result<E, DB>(m, den, v, x.x, x.y, w);
    }
    if (sets > 1) {
        float* mine = sums[grp];
#pragma unroll
        for (int k = 0; k < DB; ++k) *reinterpret_cast<f4*>(mine + 4 * q + 64 * k) = v[k];
        if (q == 0) mine[64 * DB] = m, mine[64 * DB + 1] = den;
        __syncthreads();
        for (int k = 1; k < sets && set == 0; ++k) {
            const float* o = sums[grp + k * wide];
            f4 w[DB];
#pragma unroll
            for (int e = 0; e < DB; ++e) w[e] = *reinterpret_cast<const f4*>(o + 4 * q + 64 * e);
            add_result<E, DB>(m, den, v, o[64 * DB], o[64 * DB + 1], w);
        }
    }
    if (n == 0 || set > 0) return;
    const float f = finished<E>(a, h, m, den, 16384.0f) * (1.0f / 16384.0f);
    E* op = (E*)a.out + ((int64_t)tl.row0 + r) * a.ldo + (int64_t)h * a.out_head_stride;
#pragma unroll
    for (int k = 0; k < DB; ++k)
        if (4 * q + 64 * k < dim) store4(op + 4 * q + 64 * k, v[k][0] * f, v[k][1] * f, v[k][2] * f, v[k][3] * f);
}

// Blocks that have columns, at most: tiles need not be full (full: the blocks of all rows, one after the other).
int64_t units_of(int64_t n_tiles, int64_t Hkv, int64_t cblocks, int64_t full) { return Hkv * (n_tiles * cblocks < n_tiles + full ? n_tiles * cblocks : n_tiles + full); }

// How a call is cut.  In blocks of 16 or 32 columns, the steps of everything shared out to at most two workgroups a CU (three and four: 64 single tokens 54 -> 60 .. 82 us), one for every
// eight steps (16 over 1 000 keys 15.9 us, for every four 18.6) or four of 32 columns (20 rows over 4 000 22.4, eight 23.9); from 513 tiles on a workgroup a unit.
// Or, for tiles of more than 32 columns that are work enough, blocks of 128 whose codes are converted once: from this many steps and units' costs on (us, blocks of 32 or 16 / of 128; 32
// rows of 32 heads over 2 000 keys, then 16 over 8 000): heads of 64 bf16 13.9 / 17.2, 16.7 / 16.5, of 128 17.5 / 22.2, 23.5 / 20.2, fp32 25.1 / 31.3, 37.0 / 29.8; of 192, whose
// blocks of 128 fill a CU, 17.2 / 34.1, 29.3 / 33.1 (32 requests of 32 rows over 1 000 45.5 / 43.3); of 256 28.2 / 41.2, 46.0 / 40.0.
// bf16 heads of 128 also hang on how long the units are.  64 steps and more, costs of 1 896 18.9 / 24.1, 2 144 23.7 / 21.6, 2 336 24.8 / 22.3, 2 472 22.6 / 24.6, 3 132 24.3 / 23.1, 3 264
// 24.4 / 21.8, 4 176 26.3 / 23.2; shorter ones, 2 304 19.4 / 21.3, 2 560 21.3 / 21.5, 2 880 19.6 / 20.3, 3 072 20.3 / 21.8, 3 520 11.8 / 13.1.
// Their key runs where these are too few to fill the chip twice have at least 16 steps, 8 where the blocks are less than 128 (always 8: 5 prompts of up to 600 rows, fp32, 29.0 ->
// 33.8).  Where that comes to a workgroup a CU at most, heads up to 128, it has eight waves (without / with): 216 blocks of 12 heads of 96 27.6 / 21.4, in fp32 39.0 / 32.0; few blocks
// are then cut for one a CU, not two: 64 rows of 32 heads of 64 over 16 000 keys 31.6 / 25.9, 512 of 16 of 128 over 2 000 37.5 / 31.8 (but 1 500 of 8 heads on their own, fp32, 38.4 /
// 42.7: the last rows' blocks see all keys).
Plan plan_of(bool f32, int64_t n_rows, int64_t H, int Hkv, int dim, int n_tiles, int tile_rows, int64_t longest) {
    Plan p{};
    p.per = (int)(H / Hkv);
    p.magic = p.per > 1 ? (uint32_t)(((1ull << 32) + p.per - 1) / p.per) : 0;
    const int64_t cols = (int64_t)tile_rows * p.per, steps = (longest + 63) / 64 > 0 ? (longest + 63) / 64 : 1;
    p.cols = cols <= 16 || dim > 128 ? 16 : 32;
    const int64_t small = units_of(n_tiles, Hkv, (cols + p.cols - 1) / p.cols, n_rows * p.per / p.cols) * (steps + UNIT_STEPS);
    const int64_t much = dim > 192 ? 2500 : dim > 128 ? 12500 : dim <= 64 ? 4200 : f32 ? 1400 : steps >= 64 ? 2000 : 4200;
    if (tile_rows > 1 && cols > 32 && small > much) p.cols = MANY_COLS;
    p.cblocks = (int)(cols > 1 << 30 ? 1 << 26 : (cols + p.cols - 1) / p.cols);
    int64_t units = (int64_t)n_tiles * Hkv * p.cblocks;
    p.runs = 1, p.run = 1 << 30;
    if (p.cols == MANY_COLS) {
        units = units_of(n_tiles, Hkv, p.cblocks, n_rows * p.per / MANY_COLS);
        int64_t n = units >= 512 ? 1 : units >= 128 ? (512 + units - 1) / units : (dim <= 128 ? 256 : 512) / units;
        const int64_t run = units >= 128 ? 16 : 8;                    // the least steps of one
        if (n > (steps + run - 1) / run) n = (steps + run - 1) / run;
        if (n > 1) p.run = (int)((steps + n - 1) / n), p.runs = (int)((steps + p.run - 1) / p.run);
        // (a workgroup a CU at most: eight waves each)
        p.halves = dim <= 128 && units * p.runs <= 256 && steps > 1 && (int64_t)n_tiles * Hkv * p.cblocks < 1 << 22;
    } else if (n_tiles <= SHARED_TILES && steps > 8) {
        const int each = p.cols == 32 ? 4 : 8;
        const int64_t n = (units * steps + each - 1) / each;
        p.groups = (int)(n < MAX_GROUPS ? n : MAX_GROUPS);
    }
    return p;
}
// Whether a unit's results are merged by the last of its workgroups: while columns times results stay below 256 a second launch costs more (us, two launches / one; 1 to 512 units of
// 4 columns and 1 to 63 results 17.6 / 15.0 to 194 / 190, 16 columns of 5 results 18.1 / 15.8, but of 32 16.9 / 18.3)
bool merged_in_launch(const Plan& p, int Hkv, int n_tiles, int tile_rows) {
    const int64_t cols = (int64_t)tile_rows * p.per, units = (int64_t)n_tiles * Hkv * p.cblocks;
    return (cols < p.cols ? cols : p.cols) * (p.groups / units + 1) < 256;
}
int64_t part_floats(const Plan& p, int64_t n_rows, int64_t H, int dim, int n_tiles) {
    if (p.cols == MANY_COLS) return p.runs > 1 ? n_rows * H * p.runs * (dim + 2) : 0;
    return p.groups ? head_floats(n_tiles) + 2 * (int64_t)p.groups * p.cols * (dim + 2) : 0;
}

// sizes for which a call's counts below stay inside their types
bool sizes_ok(int64_t H, int64_t Hkv, int64_t n_tiles, int64_t tile_rows) {
    return H > 0 && H <= 65535 && Hkv > 0 && H % Hkv == 0 && H / Hkv <= 2048 && n_tiles >= 0 && n_tiles < 1 << 23 && tile_rows > 0 && tile_rows * H <= 1 << 19;
}

template <typename E, int CODE, int DB>
void launch_rows(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    const dim3 grid(pl.groups ? pl.groups : a.n_tiles, pl.groups ? 1 : a.Hkv * pl.cblocks), block(256);
    if constexpr (DB <= 2)
        if (pl.cols == 32) {
            hipLaunchKernelGGL((attn_pages_rows_kernel<E, CODE, DB, 2>), grid, block, 0, stream, a, pl);
            return;
        }
    hipLaunchKernelGGL((attn_pages_rows_kernel<E, CODE, DB, 1>), grid, block, 0, stream, a, pl);
}

int merge_sets(const pcb_attn_pages_args& a, const Plan& pl) {
    const int64_t units = (int64_t)a.n_tiles * a.Hkv * pl.cblocks, results = pl.cols == MANY_COLS ? pl.runs : pl.groups / units + 1;
    return results > 32 ? 16 : results > 16 ? 8 : results > 8 ? 4 : results > 4 ? 2 : 1;
}
int64_t merge_groups(const pcb_attn_pages_args& a, const Plan& pl) {
    const int wide = 16 / merge_sets(a, pl);
    return a.n_tiles * (((int64_t)a.tile_rows * a.H + wide - 1) / wide);
}
template <typename E, int DB>
void launch_merge(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    const int sets = merge_sets(a, pl);
    hipLaunchKernelGGL((attn_pages_merge_kernel<E, DB>), dim3((unsigned)merge_groups(a, pl)), dim3(256), 0, stream, a, pl, sets);
}

template <typename E, int CODE>
int dispatch(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    if (pl.cols == MANY_COLS) {
        const int rc = pcb_attn_pages_prompt(a, pl, stream);
        if (rc != PCB_OK) return rc;
    } else if (a.dim <= 64)
        launch_rows<E, CODE, 1>(a, pl, stream);
    else if (a.dim <= 128)
        launch_rows<E, CODE, 2>(a, pl, stream);
    else if (a.dim <= 192)
        launch_rows<E, CODE, 3>(a, pl, stream);
    else
        launch_rows<E, CODE, 4>(a, pl, stream);
    if ((pl.groups && !a.counters) || pl.runs > 1) {
        if (a.dim <= 64)
            launch_merge<E, 1>(a, pl, stream);
        else if (a.dim <= 128)
            launch_merge<E, 2>(a, pl, stream);
        else
            launch_merge<E, 4>(a, pl, stream);
    }
    return pcb_check_launch("attn_pages_rows_kernel");
}

}  // namespace

PCB_EXPORT int64_t pcb_attn_pages_part(int32_t n_rows, int32_t H, int32_t Hkv, int32_t dim, int32_t n_tiles, int32_t tile_rows, int32_t longest) {
    PCB_REQUIRE(n_rows >= 0 && dim > 0 && dim <= 256 && longest >= 0 && sizes_ok(H, Hkv, n_tiles, tile_rows), PCB_ERR_ARG, "pcb_attn_pages_part: bad sizes");
    if (n_rows == 0 || n_tiles == 0) return 0;
    const int64_t a = part_floats(plan_of(false, n_rows, H, Hkv, dim, n_tiles, tile_rows, longest), n_rows, H, dim, n_tiles);
    const int64_t b = part_floats(plan_of(true, n_rows, H, Hkv, dim, n_tiles, tile_rows, longest), n_rows, H, dim, n_tiles);
    return a > b ? a : b;
}

PCB_EXPORT int pcb_attn_pages(const pcb_attn_pages_args* a, void* stream) {
    PCB_REQUIRE(a && a->struct_bytes == sizeof(pcb_attn_pages_args), PCB_ERR_ARG, "pcb_attn_pages: struct size mismatch");
    PCB_REQUIRE((a->dtype == PCB_BF16 || a->dtype == PCB_F32) && (a->code == PCB_CODE_E4M3 || a->code == PCB_CODE_INT8), PCB_ERR_ARG, "pcb_attn_pages: unknown dtype or code");
    PCB_REQUIRE(a->n_tiles >= 0 && a->tile_rows > 0 && a->n_rows >= 0 && a->n_seqs > 0 && a->max_pages > 0 && a->ld_table >= a->max_pages && a->n_pages > 0 &&
                    pcb_page_size_ok(a->page_size) && a->H > 0 && a->Hkv > 0 && a->H % a->Hkv == 0 && a->dim > 0 && a->dim <= 256 && a->dim % 16 == 0 && a->longest >= 0 &&
                    (int64_t)a->max_pages * a->page_size <= 0x7fffffff - 127,
                PCB_ERR_ARG, "pcb_attn_pages: bad sizes (pages of 16, 32, 64 or 128 tokens, heads of a multiple of 16 up to 256)");
    PCB_REQUIRE(a->scale > 0.0f && a->scale < 1e30f, PCB_ERR_ARG, "pcb_attn_pages: the score factor is a positive number");
    if (a->n_tiles == 0 || a->n_rows == 0) return PCB_OK;
    const int es = a->dtype == PCB_BF16 ? 8 : 4;
    PCB_REQUIRE(a->q && a->tiles && a->kv_len && a->table && a->kcodes && a->kscale && a->vcodes && a->vscale && a->out, PCB_ERR_ARG, "pcb_attn_pages: null pointer");
    PCB_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->kcodes | (uintptr_t)a->vcodes | (uintptr_t)a->tiles) % 16 == 0 && a->ldq % es == 0 &&
                    a->q_head_stride % es == 0 && a->ldo % es == 0 && a->out_head_stride % es == 0,
                PCB_ERR_ARG, "pcb_attn_pages: rows, heads, codes and tiles start on 16 bytes");
    PCB_REQUIRE((a->ldo != 0 || a->n_rows == 1) && (a->out_head_stride != 0 || a->H == 1), PCB_ERR_ARG, "pcb_attn_pages: results have places of their own");
    PCB_REQUIRE(sizes_ok(a->H, a->Hkv, a->n_tiles, a->tile_rows), PCB_ERR_ARG,
                "pcb_attn_pages: too many tiles, heads or tile rows (heads times tile rows up to 2^19, 2048 query heads a key head)");
    const int64_t longest = a->longest > 0 ? a->longest : (int64_t)a->max_pages * a->page_size;
    Plan p = plan_of(a->dtype == PCB_F32, a->n_rows, a->H, a->Hkv, a->dim, a->n_tiles, a->tile_rows, longest);
    if (a->window > 0 && (int64_t)a->window + a->tile_rows + 62 < longest) {   // no tile sees more keys than this: fewer runs, never more scratch
        const Plan w = plan_of(a->dtype == PCB_F32, a->n_rows, a->H, a->Hkv, a->dim, a->n_tiles, a->tile_rows, (int64_t)a->window + a->tile_rows + 62);
        if (part_floats(w, a->n_rows, a->H, a->dim, a->n_tiles) <= part_floats(p, a->n_rows, a->H, a->dim, a->n_tiles)) p = w;
    }
    p.ps = pcb_log2(a->page_size);
    // (costs are counted in 31 bits; whoever has more of them has enough units)
    if (p.groups && (int64_t)a->n_tiles * a->Hkv * p.cblocks > 0x7fffffff / ((int64_t)a->max_pages * a->page_size / 64 + 2 + UNIT_STEPS) - MAX_GROUPS) p.groups = 0;
    // (a grid is less than 2^32 threads)
    PCB_REQUIRE((int64_t)a->Hkv * p.cblocks <= 65535 && (p.cols != MANY_COLS || (int64_t)a->n_tiles * a->Hkv * p.cblocks < 1 << 23) &&
                    ((!p.groups && p.runs == 1) || merge_groups(*a, p) < 1 << 24),
                PCB_ERR_ARG, "pcb_attn_pages: too many tiles of too many heads and rows");
    PCB_REQUIRE((!p.groups && p.runs == 1) || (a->part && (uintptr_t)a->part % 16 == 0 && a->part_floats >= part_floats(p, a->n_rows, a->H, a->dim, a->n_tiles)), PCB_ERR_ARG,
                "pcb_attn_pages: shared key runs need pcb_attn_pages_part floats");
    PCB_REQUIRE((uintptr_t)a->counters % 4 == 0, PCB_ERR_ARG, "pcb_attn_pages: counters are whole numbers");
    pcb_attn_pages_args b = *a;
    if (!merged_in_launch(p, a->Hkv, a->n_tiles, a->tile_rows)) b.counters = nullptr;
    if (a->dtype == PCB_BF16)
        return a->code == PCB_CODE_E4M3 ? dispatch<bf16_t, PCB_CODE_E4M3>(b, p, (hipStream_t)stream) : dispatch<bf16_t, PCB_CODE_INT8>(b, p, (hipStream_t)stream);
    return a->code == PCB_CODE_E4M3 ? dispatch<float, PCB_CODE_E4M3>(b, p, (hipStream_t)stream) : dispatch<float, PCB_CODE_INT8>(b, p, (hipStream_t)stream);
}
