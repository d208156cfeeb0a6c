// pcb_attn_pages: causal softmax attention over keys and values held in 8 bits in pages, a power-of-two scale for each page and key head.
//
// Queries and heads of one key head are COLUMNS of a tile: column = row * (H / Hkv) + head, so a key or value is read and made a number once for all heads that
// share it.  S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16: codes of both kinds are halves exactly, a query row divided by the power of two
// of its largest element is (bf16) or is as the sum of two halves (fp32, 22 bits), and softmax weights are 11 bits (fp32: 22).  All sums are fp32.
//
// Scales never touch an operand: a page's key scale multiplies its scores.  The second product takes w = e^(s - M) vscale, M the running maximum of s + ln vscale
// over the keys a column has seen (so w <= 1 whatever the scales are, held as w 2^14 to keep halves normal down to 2^-28); the denominator sums e^(s - M) itself.
//
// A step walks 64 keys.  Lane group g (16 lanes) owns the sixteen keys 16 g .. 16 g + 15 of the step, in every role: which key a row of the first product's operand is may
// be chosen freely, so row 4 g + r of its block b is key 16 g + 4 b + r, and the lane's scores are then, in order, the keys of its operand of the second product, sixteen
// neighbouring codes of a value column, one 16-byte load.  Pages have at least 16 tokens: a lane needs one page number and one pair of scales a step.
#include "pb_pages.h"

namespace {
using namespace pcb;

constexpr float LOG2E = 1.44269504088896f;
constexpr float NEG = -__builtin_inff();

constexpr int MAX_RUNS = 256;

struct Plan {
    int ps, per, n_splits, run;        // log2 of the page size; query heads of a key head; key runs and their length in steps of 64 keys
    int cols, cblocks;                 // columns of a block, and a tile's blocks
};

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

// The lane's part of a query row as operands, sixteen neighbouring elements for each 64: two k-steps of 32.  -> the power of two that the row was divided by.
template <typename E, int DB, int PARTS>
__device__ __forceinline__ float load_query(const E* p, int dim, int g, bool live, h8 (&qf)[PARTS][2 * DB]) {
    float x[DB][16], m = 0.0f;
#pragma unroll
    for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[c][e] = 0.0f;
#pragma unroll
    for (int c = 0; c < DB; ++c) {
        const int d = 64 * c + 16 * g;
        if (live && d < dim) {
            if constexpr (sizeof(E) == 2) {
                const u32x4 a = *reinterpret_cast<const u32x4*>(p + d), b = *reinterpret_cast<const u32x4*>(p + d + 8);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[c][2 * e] = __uint_as_float(a[e] << 16), x[c][2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u);
                    x[c][8 + 2 * e] = __uint_as_float(b[e] << 16), x[c][9 + 2 * e] = __uint_as_float(b[e] & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f4 a = *reinterpret_cast<const f4*>(p + d + 4 * q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[c][4 * q + e] = a[e];
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, __builtin_fabsf(x[c][e]) < __builtin_inff() ? __builtin_fabsf(x[c][e]) : 0.0f);
    m = max4(m);
    // the row's largest element becomes 2^14 .. 2^15: what is 2^-28 of it is still a normal half
    int e2 = (int)(__float_as_uint(m) >> 23) - 127 - 14;
    e2 = e2 < -110 ? -110 : e2;
    const float inv = __uint_as_float((uint32_t)(127 - e2) << 23), unit = __uint_as_float((uint32_t)(127 + e2) << 23);
#pragma unroll
    for (int c = 0; c < DB; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = x[c][e] * inv;
            const _Float16 hi = (_Float16)y;
            qf[0][2 * c + (e >> 3)][e & 7] = hi;
            if constexpr (PARTS == 2) qf[1][2 * c + (e >> 3)][e & 7] = __builtin_fabsf(y) < __builtin_inff() ? (_Float16)(y - (float)hi) : (_Float16)0.0f;
        }
    return unit;
}

// e^x of differences of running maxima, in the units that the type keeps them in
template <typename E>
__device__ __forceinline__ float pow_of(float x) { return __builtin_amdgcn_exp2f(sizeof(E) == 4 ? x * LOG2E : x); }

// the quotient of a column: its sums under the maximum m, and the sink.  No score above -infinity: 0, but scores that are no numbers stay so
template <typename E>
__device__ __forceinline__ float finished(const pcb_attn_pages_args& a, int h, float m, float den, float num) {
    if (m == NEG) return den * 0.0f;
    if (a.sink) den += __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (a.sink[h] - m) * LOG2E : a.sink[h] * LOG2E - m);
    return num * (1.0f / 16384.0f) / den;
}

// the steps of 64 keys that some of the columns [first, last] of a tile see, and the keys that all of them do
struct Span {
    int s0, s1, all_lo, all_hi;
};
__device__ __forceinline__ Span span_of(const pcb_attn_pages_args& a, const int4& tile, int kv, int first, int last, int per) {
    const int p0 = tile.y + first / per, p1 = tile.y + last / per;
    const int end = min(kv, p1 + 1);
    int begin = a.window > 0 ? p0 - a.window + 1 : 0;
    begin = begin < 0 ? 0 : begin;
    Span s;
    s.s0 = begin >> 6, s.s1 = end > begin ? (end + 63) >> 6 : s.s0;
    s.all_lo = a.window > 0 ? p1 - a.window + 1 : 0, s.all_hi = min(kv, p0 + 1);
    return s;
}

// Sixteen scores of a lane (in units of 1 / f; -infinity: not seen) as weights of the second product: w = e^(s - M) vs 2^14 with M the running maximum of s + ln vs over the
// column's keys; l += the lane's part of sum e^(s - M); alpha: what earlier results are multiplied with.
template <typename E, int PARTS>
__device__ __forceinline__ void weights(f4 (&acc)[4], float f, float vs, float& M, float& l, float& alpha, h8 (&wf)[PARTS][2]) {
    float top = NEG;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, acc[i >> 2][i & 3]);
    const float lvs = exp_of(vs);
    top = max4(top * f + (PARTS == 2 ? lvs * 0.693147181f : lvs));    // (f > 0)
    const float M_new = fmaxf(M, top), M_use = M_new == NEG ? 0.0f : M_new;
    alpha = pow_of<E>(M - M_use);
    M = M_new;
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
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            // 2^(d log2 e) with log2 e in two parts: the error does not grow with |d|
            const float x = acc[i >> 2][i & 3] * f, d = __builtin_fmaxf(x - M_use, -200.0f);
            const float p = d * 1.44269502e+00f, rest = __builtin_fmaf(d, 1.92596303e-08f, __builtin_fmaf(d, 1.44269502e+00f, -p));
            const float q = __builtin_amdgcn_exp2f(p);
            const float e = x == NEG ? 0.0f : x == x ? __builtin_fmaf(q, rest * 6.93147182e-01f, q) : x;
            sum += e;
            const float w = e * up;
            const _Float16 top16 = (_Float16)w;
            wf[0][i >> 3][i & 7] = top16;
            wf[1][i >> 3][i & 7] = (_Float16)(w - (float)top16);
        }
    }
    l = l * alpha + sum;
}

// A workgroup: 16 NC columns of a tile and key head, a run of its keys, which the waves take step by step in turns.  A wave's keys and values go from memory straight
// into operand registers, and the next step's are asked for as soon as this one's have been multiplied: nothing crosses waves but the end.
template <typename E, int CODE, int DB, int NC, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_pages_rows_kernel(pcb_attn_pages_args a, Plan pl) {
    constexpr bool F32 = sizeof(E) == 4;
    constexpr int PARTS = F32 ? 2 : 1, NB = 4 * DB;                 // value column blocks of 16
    __shared__ float Os[NW][NB * 16][17];
    __shared__ float Ms[NW][16 * NC], Ls[NW][16 * NC];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int t = blockIdx.x, z = blockIdx.z, hk = blockIdx.y / pl.cblocks, cb = blockIdx.y % pl.cblocks;
    const int4 tile = reinterpret_cast<const int4*>(a.tiles)[t];
    const int seq = tile.x;
    if (seq < 0 || seq >= a.n_seqs) return;
    int rows = tile.z < a.tile_rows ? tile.z : a.tile_rows;
    if (tile.w < 0 || tile.y < 0 || (int64_t)tile.w + rows > a.n_rows) rows = 0;
    const int per = pl.per, col0 = cb * 16 * NC, dim = a.dim, ps = pl.ps, P = 1 << ps;
    if (col0 >= rows * per) return;
    int kv = a.kv_len[seq];
    kv = (int)min((int64_t)kv, (int64_t)a.max_pages << ps);
    const Span sp = span_of(a, tile, kv, col0, min(col0 + 16 * NC, rows * per) - 1, per);
    int s0 = sp.s0, s1 = sp.s1;
    const bool split = pl.n_splits > 1 && s1 - s0 > pl.run;           // (what one run holds is finished here)
    if (split) {
        s0 += z * pl.run;
        if (z < pl.n_splits - 1) s1 = min(s1, s0 + pl.run);
        if (s0 >= s1) return;
    } else if (z > 0) {
        return;
    }
    int lo[NC], hi[NC];                                               // a column's keys [lo, hi)
    float qs[NC];
    h8 qf[NC][PARTS][2 * DB];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int col = col0 + 16 * n + c, qr = col / per;
        const bool live = col < rows * per;
        const int pos = live ? tile.y + qr : -1, h = hk * per + (live ? col % per : 0);
        lo[n] = a.window > 0 ? pos - a.window + 1 : 0, hi[n] = min(kv, pos + 1);
        const float unit =
            load_query<E, DB, PARTS>((const E*)a.q + ((int64_t)tile.w + (live ? qr : 0)) * a.ldq + (int64_t)h * a.q_head_stride, dim, g, live, qf[n]);
        qs[n] = F32 ? unit * a.scale : unit * (a.scale * LOG2E);      // bf16: scores in units of ln 2
    }
    const int32_t* table = a.table + (int64_t)seq * a.ld_table;
    const int64_t plane = (int64_t)P * dim;
    const bool whole = dim == 64 * DB;
    float M[NC], l[NC];
    f4 o[NC][NB];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        M[n] = NEG, l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i) o[n][i] = f4{0.f, 0.f, 0.f, 0.f};
    }
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
        const int page = __shfl(pages, 4 * i + (c >> 2), 64);         // of the sixteen keys that row c of the first product's operand is one of
        const int row = ((s * 64 + 16 * (c >> 2)) & (P - 1)) + (c & 3);
        const uint8_t* p = (const uint8_t*)a.kcodes + ((int64_t)(page < 0 ? 0 : page) * a.Hkv + hk) * plane + row * dim + 16 * g;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int ch = 0; ch < DB; ++ch) {
                if (whole || 64 * ch + 16 * g < dim)
                    kr[b][ch] = *reinterpret_cast<const u32x4*>(p + 4 * b * dim + 64 * ch);
                else
                    kr[b][ch] = u32x4{0u, 0u, 0u, 0u};
            }
    };
    auto fetch_v = [&](int s, int i) {
        const int page = __shfl(pages, 4 * i + g, 64);
        const uint8_t* p = (const uint8_t*)a.vcodes + ((int64_t)(page < 0 ? 0 : page) * a.Hkv + hk) * plane + ((s * 64 + 16 * g) & (P - 1)) + c * P;
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (16 * b < dim) vr[b] = *reinterpret_cast<const u32x4*>(p + 16 * b * P);
    };
    int s = s0 + wave, i = 0;
    if (s < s1) {
        look(s);
        fetch_k(s, 0);
        fetch_v(s, 0);
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
        if (more) {
            if (i_next == 0) look(s + NW);
            fetch_k(s + NW, i_next);
        }
        // a step that all columns see whole needs no comparisons
        const bool seen = s * 64 + 64 <= sp.all_hi && s * 64 >= sp.all_lo && __all(page >= 0);
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
            weights<E, PARTS>(acc[n], qs[n] * ks, vs, M[n], l[n], alpha[n], wf[n]);
        }
        // values: codes behind the last written key are whatever the memory held, and no number times 0 is 0 for all of them
        if (!seen) {
            const int have = page < 0 ? 0 : kv - key0;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = have - 4 * e;
                    vr[b][e] &= k >= 4 ? 0xffffffffu : k <= 0 ? 0u : 0xffffffffu >> (32 - 8 * k);
                }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (16 * b >= dim) continue;
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
        if (more) fetch_v(s + NW, i_next);
        i = i_next;
    }
    // the waves' results under one maximum, sixteen columns after sixteen
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
        for (int b = 0; b < NB; ++b) {
            if (16 * b >= dim) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r) Os[wave][16 * b + 4 * g + r][c] = o[n][b][r] * back;
        }
        __syncthreads();
        const int first = col0 + 16 * n, n_live = min(16, rows * per - first);
        for (int e = tid; e < n_live * dim; e += 64 * NW) {
            const int cc = e / dim, d = e - cc * dim;
            float m = NEG, den = 0.0f, num = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) m = fmaxf(m, Ms[w][16 * n + cc]);
            const float mu = m == NEG ? 0.0f : m;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                den += Ls[w][16 * n + cc] * pow_of<E>(Ms[w][16 * n + cc] - mu);
                num += Os[w][d][cc];
            }
            const int cl = first + cc, hh = hk * per + cl % per;
            const int64_t row = (int64_t)tile.w + cl / per;
            if (split) {
                const int64_t at = (row * a.H + hh) * pl.n_splits + z;
                a.part[at * dim + d] = num;
                if (d == 0) *reinterpret_cast<float2*>(a.part + (int64_t)a.n_rows * a.H * pl.n_splits * dim + 2 * at) = float2{m, den};
            } else {
                ((E*)a.out)[row * a.ldo + (int64_t)hh * a.out_head_stride + d] = from_f32<E>(finished<E>(a, hh, m, den, num));
            }
        }
    }
}

// One workgroup a (tile, head): the key runs' results under one maximum.  The runs' factors once (a lane a run), then groups of dim / 4 threads add up every so many runs.
template <typename E>
__global__ __launch_bounds__(256) void attn_pages_merge_kernel(pcb_attn_pages_args a, Plan pl) {
    __shared__ float fac[MAX_RUNS];
    __shared__ f4 sums[256];
    __shared__ float den_s;
    const int4 tile = reinterpret_cast<const int4*>(a.tiles)[blockIdx.x];
    const int seq = tile.x, h = blockIdx.y, dim = a.dim, tid = threadIdx.x, lane = tid & 63;
    if (seq < 0 || seq >= a.n_seqs) return;
    int rows = tile.z < a.tile_rows ? tile.z : a.tile_rows;
    if (tile.w < 0 || tile.y < 0 || (int64_t)tile.w + rows > a.n_rows) rows = 0;
    int kv = a.kv_len[seq];
    kv = (int)min((int64_t)kv, (int64_t)a.max_pages << pl.ps);
    const int per = pl.per, quads = dim / 4, groups = 256 / quads, grp = tid / quads, quad = tid % quads;
    const float* ml = a.part + (int64_t)a.n_rows * a.H * pl.n_splits * dim;
    for (int r = blockIdx.z; r < rows; r += gridDim.z) {
        const int first = (r * per + h % per) / pl.cols * pl.cols;
        const Span sp = span_of(a, tile, kv, first, min(first + pl.cols, rows * per) - 1, per);   // what the row's column block walked
        if (sp.s1 - sp.s0 <= pl.run) continue;
        const int n = min(pl.n_splits, (sp.s1 - sp.s0 + pl.run - 1) / pl.run);
        const int64_t row = (int64_t)tile.w + r, at = (row * a.H + h) * pl.n_splits;
        __syncthreads();
        if (tid < 64) {
            float m = NEG;
            for (int i = lane; i < n; i += 64) m = fmaxf(m, ml[2 * (at + i)]);
            m = wave_max(m);
            const float mu = m == NEG ? 0.0f : m;
            float den = 0.0f;
            for (int i = lane; i < n; i += 64) {
                const float2 x = *reinterpret_cast<const float2*>(ml + 2 * (at + i));
                const float f = pow_of<E>(x.x - mu);
                fac[i] = f;
                den += x.y * f;
            }
            den = wave_sum(den);
            if (lane == 0) den_s = finished<E>(a, h, m, den, 16384.0f);
        }
        __syncthreads();
        f4 v = f4{0.f, 0.f, 0.f, 0.f};
        if (grp < groups)
#pragma unroll 4
            for (int i = grp; i < n; i += groups) v += *reinterpret_cast<const f4*>(a.part + (at + i) * dim + 4 * quad) * fac[i];
        sums[tid] = v;
        __syncthreads();
        if (tid < quads) {
            for (int k = 1; k < groups; ++k) v += sums[k * quads + quad];
            v *= den_s * (1.0f / 16384.0f);
            store4((E*)a.out + row * a.ldo + (int64_t)h * a.out_head_stride + 4 * quad, v[0], v[1], v[2], v[3]);
        }
    }
}

// How a call is cut.  Columns: what a tile has, in blocks of 16 or 32.  Key runs: ...
Plan plan_of(int64_t H, int Hkv, int dim, int n_tiles, int tile_rows, int64_t longest) {
    Plan p;
    p.ps = 0;
    p.per = (int)(H / Hkv);
    const int64_t cols = (int64_t)tile_rows * p.per;
    p.cols = cols <= 16 || dim > 128 ? 16 : 32;
    p.cblocks = (int)(cols > 1 << 30 ? 1 << 26 : (cols + p.cols - 1) / p.cols);
    const int64_t units = (int64_t)n_tiles * Hkv * p.cblocks, steps = (longest + 63) / 64;
    int64_t run = (units * steps + 1023) / 1024;
    run = run < 4 ? 4 : run > 16 ? 16 : run;
    if (run < units * steps / 4096) run = units * steps / 4096;
    if (run < (steps + MAX_RUNS - 1) / MAX_RUNS) run = (steps + MAX_RUNS - 1) / MAX_RUNS;
    if (steps <= 8) run = 8;
    p.run = (int)run;
    p.n_splits = (int)((steps + run - 1) / run);
    if (p.n_splits < 1) p.n_splits = 1;
    return p;
}

template <typename E, int CODE, int DB>
void launch_rows(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    const dim3 grid(a.n_tiles, a.Hkv * pl.cblocks, pl.n_splits), block(256);
    if constexpr (DB <= 2)
        if (pl.cols == 32) {
            hipLaunchKernelGGL((attn_pages_rows_kernel<E, CODE, DB, 2, 4>), grid, block, 0, stream, a, pl);
            return;
        }
    hipLaunchKernelGGL((attn_pages_rows_kernel<E, CODE, DB, 1, 4>), grid, block, 0, stream, a, pl);
}

template <typename E, int CODE>
int dispatch(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    if (a.dim <= 64)
        launch_rows<E, CODE, 1>(a, pl, stream);
    else if (a.dim <= 128)
        launch_rows<E, CODE, 2>(a, pl, stream);
    else
        launch_rows<E, CODE, 4>(a, pl, stream);
    if (pl.n_splits > 1) hipLaunchKernelGGL(attn_pages_merge_kernel<E>, dim3(a.n_tiles, a.H, a.tile_rows < 32 ? a.tile_rows : 32), dim3(256), 0, stream, a, pl);
    return pcb_check_launch("attn_pages_rows_kernel");
}

}  // namespace

PCB_EXPORT int64_t pcb_attn_pages_part(int32_t n_rows, int32_t H, int32_t Hkv, int32_t dim, int32_t n_tiles, int32_t tile_rows, int32_t longest) {
    PCB_REQUIRE(n_rows >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && dim > 0 && n_tiles >= 0 && tile_rows > 0 && longest >= 0, PCB_ERR_ARG, "pcb_attn_pages_part: bad sizes");
    if (n_rows == 0 || n_tiles == 0) return 0;
    const Plan p = plan_of(H, Hkv, dim, n_tiles, tile_rows, longest);
    return p.n_splits > 1 ? (int64_t)n_rows * H * p.n_splits * (dim + 2) : 0;
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
    const int64_t longest = a->longest > 0 ? a->longest : (int64_t)a->max_pages * a->page_size;
    Plan p = plan_of(a->H, a->Hkv, a->dim, a->n_tiles, a->tile_rows, longest);
    p.ps = pcb_log2(a->page_size);
    PCB_REQUIRE((int64_t)a->Hkv * p.cblocks <= 65535 && a->H <= 65535 && a->n_tiles < 1 << 23, PCB_ERR_ARG,
                "pcb_attn_pages: too many tiles, heads or tile rows (heads times tile rows up to 2^20)");
    PCB_REQUIRE(p.n_splits == 1 || (a->part && (uintptr_t)a->part % 16 == 0 && a->part_floats >= (int64_t)a->n_rows * a->H * p.n_splits * (a->dim + 2)), PCB_ERR_ARG,
                "pcb_attn_pages: key runs need pcb_attn_pages_part floats");
    if (a->dtype == PCB_BF16)
        return a->code == PCB_CODE_E4M3 ? dispatch<bf16_t, PCB_CODE_E4M3>(*a, p, (hipStream_t)stream) : dispatch<bf16_t, PCB_CODE_INT8>(*a, p, (hipStream_t)stream);
    return a->code == PCB_CODE_E4M3 ? dispatch<float, PCB_CODE_E4M3>(*a, p, (hipStream_t)stream) : dispatch<float, PCB_CODE_INT8>(*a, p, (hipStream_t)stream);
}
