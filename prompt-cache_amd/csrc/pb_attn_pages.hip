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

struct Plan {
    int ps, per, n_splits, run;        // log2 of the page size; query heads of a key head; key runs and their length in steps of 64 keys
    int cblocks;                       // column blocks of a tile
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

// what a wave's step needs of its sixteen keys' page
struct KeyPage {
    int page;                          // -1: none
    float ks, vs;
};

template <typename E, int CODE, int DB, int NW>
__global__ __launch_bounds__(64 * NW) void attn_pages_rows_kernel(pcb_attn_pages_args a, Plan pl) {
    constexpr int PARTS = sizeof(E) == 4 ? 2 : 1, NB = 4 * DB;      // value column blocks of 16
    __shared__ float Os[NW][NB * 16][17];
    __shared__ float Ms[NW][16], Ls[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int t = blockIdx.x, z = blockIdx.z, hk = blockIdx.y / pl.cblocks, cb = blockIdx.y % pl.cblocks;
    const int4 tile = reinterpret_cast<const int4*>(a.tiles)[t];
    const int seq = tile.x;
    if (seq < 0 || seq >= a.n_seqs) return;
    int rows = tile.z < a.tile_rows ? tile.z : a.tile_rows;
    if (tile.w < 0 || tile.y < 0 || (int64_t)tile.w + rows > a.n_rows) rows = 0;
    const int per = pl.per, col0 = cb * 16, dim = a.dim, ps = pl.ps, P = 1 << ps;
    if (col0 >= rows * per) return;
    const int col = col0 + c, qr = col / per, h = hk * per + col % per;
    const bool live = col < rows * per;
    const int last_col = min(col0 + 15, rows * per - 1);
    const int first_pos = tile.y + col0 / per, last_pos = tile.y + last_col / per, pos = live ? tile.y + qr : -1;
    int kv = a.kv_len[seq];
    kv = (int)min((int64_t)kv, (int64_t)a.max_pages << ps);
    const int end = min(kv, last_pos + 1);                            // keys [begin, end) are seen by some column
    int begin = a.window > 0 ? first_pos - a.window + 1 : 0;
    begin = begin < 0 ? 0 : begin;
    const int lo = a.window > 0 ? pos - a.window + 1 : 0, hi = min(kv, pos + 1);   // this column's keys [lo, hi)
    int s0 = begin >> 6, s1 = end > begin ? (end + 63) >> 6 : s0;     // steps of 64 keys
    const int all = s1 - s0;
    const bool split = pl.n_splits > 1 && all > pl.run;               // (a tile of one run is finished here)
    if (split) {
        s0 += z * pl.run;
        if (z < pl.n_splits - 1) s1 = min(s1, s0 + pl.run);
        if (s0 >= s1) return;
    } else if (z > 0) {
        return;
    }
    const int64_t qrow = (int64_t)tile.w + (live ? qr : 0);
    h8 qf[PARTS][2 * DB];
    const float unit = load_query<E, DB, PARTS>((const E*)a.q + qrow * a.ldq + (int64_t)(live ? h : hk * per) * a.q_head_stride, dim, g, live, qf);
    const float qs = sizeof(E) == 4 ? unit * a.scale : unit * (a.scale * LOG2E);   // bf16: scores in units of ln 2

    const int32_t* table = a.table + (int64_t)seq * a.ld_table;
    const int64_t plane = (int64_t)P * dim;
    float M = NEG, l = 0.0f;
    f4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};

    for (int s = s0 + wave; s < s1; s += NW) {
        // the page of this lane's sixteen keys, and (first product's operand) of the sixteen that row c >> 2 belongs to
        const int key0 = s * 64 + 16 * g;
        int page = key0 < kv ? table[key0 >> ps] : -1;
        page = page >= 0 && page < a.n_pages ? page : -1;
        const int64_t ph = (int64_t)(page < 0 ? 0 : page) * a.Hkv + hk;
        const float ks = page < 0 ? 1.0f : a.kscale[ph], vs = page < 0 ? 1.0f : a.vscale[ph];
        const int kpage = __shfl(page, 16 * (c >> 2), 64);
        const int krow0 = ((s * 64 + 16 * (c >> 2)) & (P - 1)) + (c & 3);
        const uint8_t* kp = (const uint8_t*)a.kcodes + ((int64_t)(kpage < 0 ? 0 : kpage) * a.Hkv + hk) * plane + (int64_t)krow0 * dim + 16 * g;
        f4 acc[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            acc[b] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ch = 0; ch < DB; ++ch) {
                u32x4 w = u32x4{0u, 0u, 0u, 0u};
                if (64 * ch + 16 * g < dim) w = *reinterpret_cast<const u32x4*>(kp + (int64_t)4 * b * dim + 64 * ch);
                const h8 k0 = half8<CODE>(u32x2{w[0], w[1]}), k1 = half8<CODE>(u32x2{w[2], w[3]});
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[p][2 * ch], acc[b], 0, 0, 0);
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[p][2 * ch + 1], acc[b], 0, 0, 0);
                }
            }
        }
        // scores; what a column does not see is -infinity
        const float f = qs * ks, lvs = exp_of(vs);
        float x[16], top = NEG;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = key0 + i;
            x[i] = page >= 0 && key >= lo && key < hi ? acc[i >> 2][i & 3] * f : NEG;
            top = fmaxf(top, x[i]);
        }
        top = max4(top + (sizeof(E) == 4 ? lvs * 0.693147181f : lvs));
        const float M_new = fmaxf(M, top);
        const float M_use = M_new == NEG ? 0.0f : M_new;
        float alpha, sum = 0.0f;
        if constexpr (sizeof(E) == 4)
            alpha = __builtin_amdgcn_exp2f((M - M_use) * LOG2E);
        else
            alpha = __builtin_amdgcn_exp2f(M - M_use);
        const float up = vs * 16384.0f;
        h8 wf[PARTS][2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float e;
            if constexpr (sizeof(E) == 4) {
                // 2^(d log2 e) with log2 e in two parts: the error does not grow with |d|
                const float d = __builtin_fmaxf(x[i] - M_use, -200.0f);
                const float p = d * 1.44269502e+00f, rest = __builtin_fmaf(d, 1.92596303e-08f, __builtin_fmaf(d, 1.44269502e+00f, -p));
                const float q = __builtin_amdgcn_exp2f(p);
                e = x[i] == NEG ? 0.0f : x[i] == x[i] ? __builtin_fmaf(q, rest * 6.93147182e-01f, q) : x[i];
            } else {
                e = __builtin_amdgcn_exp2f(x[i] - M_use);
            }
            sum += e;
            const float w = e * up;
            const _Float16 hi16 = (_Float16)w;
            wf[0][i >> 3][i & 7] = hi16;
            if constexpr (PARTS == 2) wf[1][i >> 3][i & 7] = (_Float16)(w - (float)hi16);
        }
        l = l * alpha + sum;
        M = M_new;
        // values: codes behind the last written key are whatever the memory held, and no number times 0 is 0 for all of them
        const int have = page < 0 ? 0 : kv - key0;
        const uint8_t* vp = (const uint8_t*)a.vcodes + ph * plane + (key0 & (P - 1));
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (16 * i >= dim) break;
            u32x4 w = *reinterpret_cast<const u32x4*>(vp + (int64_t)(16 * i + c) * P);
            if (have < 16) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = have - 4 * e;
                    w[e] &= n >= 4 ? 0xffffffffu : n <= 0 ? 0u : 0xffffffffu >> (32 - 8 * n);
                }
            }
            const h8 v0 = half8<CODE>(u32x2{w[0], w[1]}), v1 = half8<CODE>(u32x2{w[2], w[3]});
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i][r] *= alpha;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, wf[p][0], o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, wf[p][1], o[i], 0, 0, 0);
            }
        }
    }
    // the waves' results under one maximum
    l = sum4(l);
    if (g == 0) Ms[wave][c] = M, Ls[wave][c] = l;
    __syncthreads();
    float top = NEG;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, Ms[w][c]);
    const float top_use = top == NEG ? 0.0f : top;
    const float back = __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (M - top_use) * LOG2E : M - top_use);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        if (16 * i >= dim) break;
#pragma unroll
        for (int r = 0; r < 4; ++r) Os[wave][16 * i + 4 * g + r][c] = o[i][r] * back;
    }
    __syncthreads();
    const int n_live = min(16, rows * per - col0);
    for (int i = tid; i < n_live * dim; i += 64 * NW) {
        const int cc = i / dim, d = i - cc * dim;
        float m = NEG, den = 0.0f, num = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, Ms[w][cc]);
        const float mu = m == NEG ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            den += Ls[w][cc] * __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (Ms[w][cc] - mu) * LOG2E : Ms[w][cc] - mu);
            num += Os[w][d][cc];
        }
        const int cl = col0 + cc, hh = hk * per + cl % per;
        const int64_t row = (int64_t)tile.w + cl / per;
        if (split) {
            float* pp = a.part + ((row * a.H + hh) * pl.n_splits + z) * (dim + 2);
            pp[d] = num;
            if (d == 0) pp[dim] = m, pp[dim + 1] = den;
        } else {
            if (a.sink && m != NEG) den += __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (a.sink[hh] - mu) * LOG2E : a.sink[hh] * LOG2E - mu);
            const float v = m == NEG ? den * 0.0f : num * (1.0f / 16384.0f) / den;   // (no score above -infinity: 0, but scores that are no numbers stay so)
            ((E*)a.out)[row * a.ldo + (int64_t)hh * a.out_head_stride + d] = from_f32<E>(v);
        }
    }
}

// One workgroup a (tile, head): the key runs' results under one maximum.
template <typename E>
__global__ __launch_bounds__(256) void attn_pages_merge_kernel(pcb_attn_pages_args a, Plan pl) {
    const int4 tile = reinterpret_cast<const int4*>(a.tiles)[blockIdx.x];
    const int seq = tile.x, h = blockIdx.y, dim = a.dim;
    if (seq < 0 || seq >= a.n_seqs) return;
    int rows = tile.z < a.tile_rows ? tile.z : a.tile_rows;
    if (tile.w < 0 || tile.y < 0 || (int64_t)tile.w + rows > a.n_rows) rows = 0;
    int kv = a.kv_len[seq];
    kv = (int)min((int64_t)kv, (int64_t)a.max_pages << pl.ps);
    const int per = pl.per;
    for (int r = 0; r < rows; ++r) {
        // the same steps that the row's column block walked
        const int col0 = (r * per + h % per) / 16 * 16, last_col = min(col0 + 15, rows * per - 1);
        const int first_pos = tile.y + col0 / per, last_pos = tile.y + last_col / per;
        const int end = min(kv, last_pos + 1);
        int begin = a.window > 0 ? first_pos - a.window + 1 : 0;
        begin = begin < 0 ? 0 : begin;
        const int s0 = begin >> 6, s1 = end > begin ? (end + 63) >> 6 : s0, all = s1 - s0;
        if (all <= pl.run) continue;
        const int n = min(pl.n_splits, (all + pl.run - 1) / pl.run);
        const int64_t row = (int64_t)tile.w + r;
        const float* pp = a.part + (row * a.H + h) * pl.n_splits * (dim + 2);
        float m = NEG;
        for (int i = 0; i < n; ++i) m = fmaxf(m, pp[(int64_t)i * (dim + 2) + dim]);
        const float mu = m == NEG ? 0.0f : m;
        float den = a.sink && m != NEG ? __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (a.sink[h] - mu) * LOG2E : a.sink[h] * LOG2E - mu) : 0.0f;
        for (int i = 0; i < n; ++i) {
            const float* q = pp + (int64_t)i * (dim + 2) + dim;
            den += q[1] * __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (q[0] - mu) * LOG2E : q[0] - mu);
        }
        for (int d = threadIdx.x; d < dim; d += 256) {
            float num = 0.0f;
            for (int i = 0; i < n; ++i) {
                const float* q = pp + (int64_t)i * (dim + 2);
                num += q[d] * __builtin_amdgcn_exp2f(sizeof(E) == 4 ? (q[dim] - mu) * LOG2E : q[dim] - mu);
            }
            const float v = m == NEG ? den * 0.0f : num * (1.0f / 16384.0f) / den;   // (no score above -infinity: 0, but scores that are no numbers stay so)
            ((E*)a.out)[row * a.ldo + (int64_t)h * a.out_head_stride + d] = from_f32<E>(v);
        }
    }
}

// key runs: enough workgroups for the chip, none shorter than a step for each wave
Plan plan_of(int64_t H, int Hkv, int n_tiles, int tile_rows, int64_t longest) {
    Plan p;
    p.ps = 0;
    p.per = (int)(H / Hkv);
    const int64_t cols = (int64_t)tile_rows * p.per;
    p.cblocks = (int)(cols > 1 << 30 ? 1 << 26 : (cols + 15) / 16);
    const int64_t units = (int64_t)n_tiles * Hkv * p.cblocks, steps = (longest + 63) / 64;
    int64_t n = (1024 + units - 1) / units;
    if (n > (steps + 3) / 4) n = (steps + 3) / 4;
    if (n > 128) n = 128;
    if (n < 1) n = 1;
    p.run = (int)((steps + n - 1) / n);
    if (p.run < 1) p.run = 1;
    p.n_splits = (int)((steps + p.run - 1) / p.run);
    if (p.n_splits < 1) p.n_splits = 1;
    return p;
}

template <typename E, int CODE>
int dispatch(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    const dim3 grid(a.n_tiles, a.Hkv * pl.cblocks, pl.n_splits), block(256);
    if (a.dim <= 64)
        hipLaunchKernelGGL((attn_pages_rows_kernel<E, CODE, 1, 4>), grid, block, 0, stream, a, pl);
    else if (a.dim <= 128)
        hipLaunchKernelGGL((attn_pages_rows_kernel<E, CODE, 2, 4>), grid, block, 0, stream, a, pl);
    else
        hipLaunchKernelGGL((attn_pages_rows_kernel<E, CODE, 4, 4>), grid, block, 0, stream, a, pl);
    if (pl.n_splits > 1) hipLaunchKernelGGL(attn_pages_merge_kernel<E>, dim3(a.n_tiles, a.H), dim3(256), 0, stream, a, pl);
    return pcb_check_launch("attn_pages_rows_kernel");
}

}  // namespace

PCB_EXPORT int64_t pcb_attn_pages_part(int32_t n_rows, int32_t H, int32_t Hkv, int32_t dim, int32_t n_tiles, int32_t tile_rows, int32_t longest) {
    PCB_REQUIRE(n_rows >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && dim > 0 && n_tiles >= 0 && tile_rows > 0 && longest >= 0, PCB_ERR_ARG, "pcb_attn_pages_part: bad sizes");
    if (n_rows == 0 || n_tiles == 0) return 0;
    const Plan p = plan_of(H, Hkv, n_tiles, tile_rows, longest);
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
    Plan p = plan_of(a->H, a->Hkv, a->n_tiles, a->tile_rows, longest);
    p.ps = pcb_log2(a->page_size);
    PCB_REQUIRE((int64_t)a->Hkv * p.cblocks <= 65535 && a->H <= 65535 && a->n_tiles < 1 << 23, PCB_ERR_ARG,
                "pcb_attn_pages: too many tiles, heads or tile rows (heads times tile rows up to 2^20)");
    PCB_REQUIRE(p.n_splits == 1 || (a->part && (uintptr_t)a->part % 16 == 0 && a->part_floats >= (int64_t)a->n_rows * a->H * p.n_splits * (a->dim + 2)), PCB_ERR_ARG,
                "pcb_attn_pages: key runs need pcb_attn_pages_part floats");
    if (a->dtype == PCB_BF16)
        return a->code == PCB_CODE_E4M3 ? dispatch<bf16_t, PCB_CODE_E4M3>(*a, p, (hipStream_t)stream) : dispatch<bf16_t, PCB_CODE_INT8>(*a, p, (hipStream_t)stream);
    return a->code == PCB_CODE_E4M3 ? dispatch<float, PCB_CODE_E4M3>(*a, p, (hipStream_t)stream) : dispatch<float, PCB_CODE_INT8>(*a, p, (hipStream_t)stream);
}
