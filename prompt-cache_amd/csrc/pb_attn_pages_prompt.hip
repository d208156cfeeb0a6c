// pcb_attn_pages for tiles of many columns (pb_attn_pages.hip: what a column, a step and a scale are): prompts behind cached prefixes, long questions.
//
// One workgroup = 128 columns of a tile and one key head, 32 a wave, over the keys they see (or a run of these, where the tiles are too few to fill the chip).  A step's 64 keys and
// values become halves once for all four waves: codes go memory -> registers a step ahead, are converted and written to one of two LDS images while the other one is multiplied.
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_f16: a lane owns one column, its 32 scores of a step are its own operand of the second product (row 8 i + 4 h + j of the
// first product's operand is key 16 (i / 2) + 8 h + 4 (i % 2) + j of 32, so lane half h holds keys 16 m + 8 h .. + 7), and a column's maximum is one exchange between two lanes.
//
// Bound by the two products and the softmax between them: a step of 64 keys is 2 x 16 MFMA and 32 exponentials a wave of heads of 128.  Measured: 3 989 rows of 32 heads of 128 over
// 8 heads' prefixes of 4 096 .. 6 200 keys, bf16, 425 GFLOP: 489 us = 0.87 PFLOP/s, where a large fp16 product of the library reaches 1.12 (both lower the clock); fp32 (two halves
// of a query and of a weight under codes that are whole, so twice the products) 864 us.  5 prompts of 1 877 rows of 15 heads of 96 under a window of 333, fp32: 29 us, of which a block's
// steps, at most 7, take 2.2 each and what is around them 15 (a window of 1: 17.3; in bf16 10.8): 230 workgroups of four waves, one a CU, have nothing beside a wave that waits.
//
// LDS rows are 16 bytes longer than their 32 ND halves of a key, or 64 keys of a value column: the sixteen lanes that are served at once fall on all banks.
#include "pb_attn_pages.h"

namespace {
using namespace pcb;

typedef float f16v __attribute__((ext_vector_type(16)));

// the larger, or the sum, of a lane's number and that of the lane 32 further
__device__ __forceinline__ float max2(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum2(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float lane_of(float v, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)); }

// ND: value columns (and key elements) in blocks of 32.  KS = 2: eight waves, of which the second four take every other step with images of their own, so that a CU that has one
// workgroup still has two waves a SIMD, one multiplying while the other one is at its softmax; their results meet in LDS.
template <typename E, int CODE, int ND, int KS>
__global__ __launch_bounds__(256 * KS, KS == 1 && sizeof(E) == 2 && ND <= 6 ? 2 : 1) void attn_pages_prompt_kernel(pcb_attn_pages_args a, Plan pl) {
    constexpr bool F32 = sizeof(E) == 4;
    constexpr int PARTS = F32 ? 2 : 1, KK = 2 * ND;                   // k-steps of 16 of the first product
    constexpr int KLD = 32 * ND + 8, VLD = 72, PIECES = 128 * ND, NP = (PIECES + 255) / 256;   // sixteen-byte pieces of a step's keys, and of its values; of each a thread's
    constexpr int OLD = 32 * ND + 4;                                  // a column's sums, where the two halves of the waves meet
    // (bf16 heads of 192: one image, and so two workgroups a CU: 2 000 rows of 32 heads over 4 000 keys 391 -> 305 us; 256 elements' sums and queries leave no registers for two)
    constexpr int BUFS = !F32 && ND == 6 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) _Float16 images[KS][BUFS][64 * KLD + 32 * ND * VLD];
    const int tid = threadIdx.x & 255, kg = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, c = lane & 31;
    const int hk = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv, cb = rest % pl.cblocks, t = a.n_tiles - 1 - rest / pl.cblocks;   // (a prompt's last tiles, which see most keys, first)
    const int dim = a.dim, ps = pl.ps, P = 1 << ps, per = pl.per;
    Tile tl = tile_of(a, t, ps);
    const int cols = tl.rows * per, col0 = cb * MANY_COLS;
    if (col0 >= cols) return;
    const int kv = tl.kv;
    tl = rows_of(a, tl, row_of(pl, col0), row_of(pl, min(col0 + MANY_COLS, cols) - 1));
    int s0 = tl.s0, s1 = tl.s1;
    const bool split = pl.runs > 1 && s1 - s0 > pl.run;
    if (split) {
        s0 += (int)blockIdx.y * pl.run;
        if ((int)blockIdx.y < pl.runs - 1) s1 = min(s1, s0 + pl.run);
        if (s0 >= s1) return;
    } else if (blockIdx.y > 0) {
        return;
    }
    const int32_t* table = a.table + (int64_t)tl.seq * a.ld_table;
    const int64_t plane = (int64_t)P * dim;
    // pages and scales of sixteen steps at once: lane 4 i + k those of step i's keys 16 k ..
    int pages = -1;
    float kss = 1.0f, vss = 1.0f;
    auto look = [&](int s) {
        const int key = (s + (lane >> 2) * KS) * 64 + 16 * (lane & 3);
        pages = s + (lane >> 2) * KS < s1 && key < kv ? table[key >> ps] : -1;
        pages = pages >= 0 && pages < a.n_pages ? pages : -1;
        const int64_t ph = (int64_t)(pages < 0 ? 0 : pages) * a.Hkv + hk;
        kss = pages < 0 ? 1.0f : a.kscale[ph], vss = pages < 0 ? 1.0f : a.vscale[ph];
    };
    // staging: thread t takes pieces t, t + 256, .. of the step's keys (2 ND a row) and of its value columns (four a column, the same sixteen keys each time)
    const int vq = tid & 3;
    u32x4 kr[NP], vr[NP];
    auto fetch = [&](int s, int i) {
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int piece = min(n * 256 + tid, PIECES - 1), row = piece / (2 * ND), ch = piece % (2 * ND);
            const int page = __shfl(pages, 4 * i + (row >> 4), 64);
            const uint8_t* p = (const uint8_t*)a.kcodes + ((int64_t)(page < 0 ? 0 : page) * a.Hkv + hk) * plane + ((s * 64 + row) & (P - 1)) * dim;
            kr[n] = *reinterpret_cast<const u32x4*>(p + 16 * min(ch, dim / 16 - 1));
        }
        const int page = __shfl(pages, 4 * i + vq, 64);
        const uint8_t* p = (const uint8_t*)a.vcodes + ((int64_t)(page < 0 ? 0 : page) * a.Hkv + hk) * plane + ((s * 64 + 16 * vq) & (P - 1));
#pragma unroll
        for (int n = 0; n < NP; ++n) vr[n] = *reinterpret_cast<const u32x4*>(p + min(n * 64 + (tid >> 2), dim - 1) * P);
        // values behind the last written key are whatever the memory held, and no number times 0 is 0 for all of them
        const int have = page < 0 ? 0 : kv - (s * 64 + 16 * vq);
        if (have < 16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = have - 4 * e;
                const uint32_t keep = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : 0xffffffffu >> (32 - 8 * k);
#pragma unroll
                for (int n = 0; n < NP; ++n) vr[n][e] &= keep;
            }
        }
    };
    auto stage = [&](int buf) {
        _Float16 *Ks = images[kg][buf], *Vs = Ks + 64 * KLD;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            if (PIECES % 256 && n * 256 + tid >= PIECES) break;
            const int row = (n * 256 + tid) / (2 * ND), ch = (n * 256 + tid) % (2 * ND);
            _Float16* k = Ks + row * KLD + 16 * ch;
            *reinterpret_cast<h8*>(k) = half8<CODE>(u32x2{kr[n][0], kr[n][1]});
            *reinterpret_cast<h8*>(k + 8) = half8<CODE>(u32x2{kr[n][2], kr[n][3]});
            _Float16* v = Vs + (n * 64 + (tid >> 2)) * VLD + 16 * vq;
            *reinterpret_cast<h8*>(v) = half8<CODE>(u32x2{vr[n][0], vr[n][1]});
            *reinterpret_cast<h8*>(v + 8) = half8<CODE>(u32x2{vr[n][2], vr[n][3]});
        }
    };
    int i = 0;
    if (s0 + kg < s1) {
        look(s0 + kg);
        fetch(s0 + kg, 0);
    }
    // this lane's column
    const int col = col0 + 32 * wave + c;
    const bool live = col < cols;
    const int qr = live ? row_of(pl, col) : 0, h = hk * per + (live ? col - qr * per : 0), pos = live ? tl.pos + qr : -1;
    const int lo = a.window > 0 ? pos - a.window + 1 : 0, hi = min(kv, pos + 1);
    // keys that all, and that some of the wave's columns see
    const int wc0 = col0 + 32 * wave, wc1 = min(wc0 + 32, cols) - 1;
    const bool wave_live = wc0 < cols;
    const int p0 = tl.pos + row_of(pl, wave_live ? wc0 : 0), p1 = tl.pos + row_of(pl, wave_live ? wc1 : 0);
    const int all_lo = a.window > 0 ? p1 - a.window + 1 : 0, all_hi = wc0 + 32 <= cols ? min(kv, p0 + 1) : 0;
    const int any_lo = a.window > 0 ? p0 - a.window + 1 : 0, any_hi = wave_live ? min(kv, p1 + 1) : 0;
    h8 qf[PARTS][KK];
    float qs;
    {
        const E* q = (const E*)a.q + ((int64_t)tl.row0 + qr) * a.ldq + (int64_t)h * a.q_head_stride;
        float x[KK][8], m = 0.0f;
#pragma unroll
        for (int k = 0; k < KK; ++k) {
            Frag<E> f;
            zero8(f);
            if (live && 16 * k < dim) f = load8(q + 16 * k + 8 * hh);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[k][e] = at8(f, e);
                m = fmaxf(m, __builtin_fabsf(x[k][e]) < __builtin_inff() ? __builtin_fabsf(x[k][e]) : 0.0f);
            }
        }
        // divided by a power of two, the row's largest element is 2^14 .. 2^15: what is 2^-28 of it is still a normal half
        m = max2(m);
        int e2 = (int)(__float_as_uint(m) >> 23) - 127 - 14;
        e2 = e2 < -110 ? -110 : e2;
        const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
        qs = __uint_as_float((uint32_t)(127 + e2) << 23) * (F32 ? a.scale : a.scale * LOG2E);
#pragma unroll
        for (int k = 0; k < KK; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = x[k][e] * inv;
                const _Float16 top = (_Float16)y;
                qf[0][k][e] = top;
                if constexpr (PARTS == 2) qf[1][k][e] = __builtin_fabsf(y) < __builtin_inff() ? (_Float16)(y - (float)top) : (_Float16)0.0f;
            }
    }
    float M = NEG, l = 0.0f;
    f16v o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
    if (s0 + kg < s1) stage(0);
    const int krow = (c >> 4) * 16 + ((c >> 2) & 1) * 8 + ((c >> 3) & 1) * 4 + (c & 3);   // the key of 32 that row c of the first product's operand is
    int buf = 0;
    for (int s = s0 + kg; s - kg < s1; s += KS) {
        // the step's scales, before `look` takes the next ones' place
        float ks[4], vs[4];
        bool whole = s * 64 + 64 <= all_hi && s * 64 >= all_lo;
        int page_ok = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            ks[q] = lane_of(kss, 4 * i + q), vs[q] = lane_of(vss, 4 * i + q);
            page_ok |= (__builtin_amdgcn_readlane(pages, 4 * i + q) >= 0 ? 1 : 0) << q;
        }
        whole = whole && page_ok == 15;
        const bool more = s + KS < s1;
        __syncthreads();                                              // the step's image is written, the other one read
        i = (i + 1) & 15;
        if (more) {
            if (i == 0) look(s + KS);
            fetch(s + KS, i);
        }
        if ((KS == 1 || s < s1) && s * 64 < any_hi && s * 64 + 64 > any_lo) {
            f16v acc[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[b][e] = 0.0f;
                const _Float16* k = &images[kg][buf][(32 * b + krow) * KLD + 8 * hh];
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const h8 f = *reinterpret_cast<const h8*>(k + 16 * kk);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qf[p][kk], acc[b], 0, 0, 0);
                }
            }
            if (!whole) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = s * 64 + 32 * b + 16 * (e >> 3) + 8 * hh + (e & 7);
                        if (!(key >= lo && key < hi && (page_ok >> (2 * b + (e >> 3)) & 1))) acc[b][e] = NEG;
                    }
            }
            float f[4], top = NEG;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f[q] = score_unit(qs, ks[q]);
                float m = acc[q >> 1][8 * (q & 1)];
#pragma unroll
                for (int e = 1; e < 8; ++e) m = fmaxf(m, acc[q >> 1][8 * (q & 1) + e]);
                top = fmaxf(top, __builtin_fmaf(m, f[q], F32 ? exp_of(vs[q]) * 0.693147181f : exp_of(vs[q])));
            }
            top = max2(top);
            const float M_new = fmaxf(M, top);
            float M_use = M_new == NEG ? 0.0f : M_new;
            const float alpha = pow_of<E>(M - M_use);
            if (__builtin_expect(__builtin_fabsf(M_use) > FAR, 0)) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        acc[q >> 1][8 * (q & 1) + e] = above(acc[q >> 1][8 * (q & 1) + e], f[q], F32 ? exp_of(vs[q]) * 0.693147181f : exp_of(vs[q]), M_use);
                    f[q] = 1.0f;
                }
                M_use = 0.0f;
            }
            h8 wf[PARTS][4];
            float sum = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float part = 0.0f;
                if constexpr (!F32) {
                    const float off = exp_of(vs[q]) + 14.0f - M_use;  // vscale and 2^14 inside the exponent, out of the sum again
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[q >> 1][8 * (q & 1) + e], f[q], off));
                        part += w;
                        wf[0][q][e] = (_Float16)w;
                    }
                    sum = __builtin_fmaf(part, inv_pow2(vs[q]) * (1.0f / 16384.0f), sum);
                } else {
                    const float up = vs[q] * 16384.0f;
                    float scores = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float s1 = acc[q >> 1][8 * (q & 1) + e], ex = exp_of_score(s1, f[q], M_use);
                        scores += s1;
                        part += ex;
                        _Float16 hi, lo;
                        two_halves(ex * up, hi, lo);
                        wf[0][q][e] = hi, wf[1][q][e] = lo;
                    }
                    sum += or_not(part, scores);
                }
            }
            l = l * alpha + sum;
            if (!__all(M_new == M)) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
            }
            M = M_new;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const h8 x = *reinterpret_cast<const h8*>(&images[kg][buf][64 * KLD + (32 * d + c) * VLD + 8 * hh + 16 * m]);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, wf[p][m], o[d], 0, 0, 0);
                }
            }
        }
        if (BUFS == 1) __syncthreads();                               // (the image has been read)
        if (more) stage(BUFS == 1 ? 0 : buf ^ 1);
        if (BUFS == 2) buf ^= 1;
    }
    l = sum2(l);
    if constexpr (KS == 2) {
        float* sums = reinterpret_cast<float*>(&images[0][0][0]) + (32 * wave + c) * (OLD + 2);
        static_assert(128 * (OLD + 2) * 4 <= (int)sizeof(images), "the sums of 128 columns in the images' place");
        __syncthreads();                                              // (all images have been multiplied)
        if (kg == 1) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) sums[32 * d + 8 * (e >> 2) + 4 * hh + (e & 3)] = o[d][e];
            if (hh == 0) sums[OLD] = M, sums[OLD + 1] = l;
        }
        __syncthreads();
        if (kg == 1) return;
        const float M1 = sums[OLD], top = fmaxf(M, M1), use = top == NEG ? 0.0f : top, x = pow_of<E>(M - use), y = pow_of<E>(M1 - use);
        M = top, l = l * x + sums[OLD + 1] * y;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = o[d][e] * x + sums[32 * d + 8 * (e >> 2) + 4 * hh + (e & 3)] * y;
    }
    if (!live) return;
    E* op = (E*)a.out + ((int64_t)tl.row0 + qr) * a.ldo + (int64_t)h * a.out_head_stride;
    const int64_t at_part = (((int64_t)tl.row0 + qr) * a.H + h) * pl.runs + blockIdx.y;
    float* pp = a.part + at_part * dim;
    const float f = split ? 1.0f : finished<E>(a, h, M, l, 16384.0f) * (1.0f / 16384.0f);
    if (split && hh == 0) *reinterpret_cast<float2*>(a.part + (int64_t)a.n_rows * a.H * pl.runs * dim + 2 * at_part) = float2{M, l};
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = 32 * d + 8 * q + 4 * hh;
            if (at >= dim) continue;
            if (split)
                *reinterpret_cast<f4*>(pp + at) = f4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
            else
                store4(op + at, o[d][4 * q] * f, o[d][4 * q + 1] * f, o[d][4 * q + 2] * f, o[d][4 * q + 3] * f);
        }
}

template <typename E, int CODE, int ND, int KS>
void launch_one(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)a.n_tiles * a.Hkv * pl.cblocks), pl.runs);
    hipLaunchKernelGGL((attn_pages_prompt_kernel<E, CODE, ND, KS>), grid, dim3(256 * KS), 0, stream, a, pl);
}
template <typename E, int CODE>
int launch(const pcb_attn_pages_args& a, const Plan& pl, hipStream_t stream) {
    const int blocks = (a.dim + 31) / 32;
    if (pl.halves && blocks <= 2)
        launch_one<E, CODE, 2, 2>(a, pl, stream);
    else if (pl.halves && blocks == 3)
        launch_one<E, CODE, 3, 2>(a, pl, stream);
    else if (pl.halves && blocks == 4)
        launch_one<E, CODE, 4, 2>(a, pl, stream);
    else if (blocks <= 2)
        launch_one<E, CODE, 2, 1>(a, pl, stream);
    else if (blocks == 3)
        launch_one<E, CODE, 3, 1>(a, pl, stream);
    else if (blocks == 4)
        launch_one<E, CODE, 4, 1>(a, pl, stream);
    else if (blocks <= 6)
        launch_one<E, CODE, 6, 1>(a, pl, stream);
    else
        launch_one<E, CODE, 8, 1>(a, pl, stream);
    return pcb_check_launch("attn_pages_prompt_kernel");
}

}  // namespace

int pcb_attn_pages_prompt(const pcb_attn_pages_args& a, const pcb::Plan& pl, hipStream_t stream) {
    if (a.dtype == PCB_BF16) return a.code == PCB_CODE_E4M3 ? launch<pcb::bf16_t, PCB_CODE_E4M3>(a, pl, stream) : launch<pcb::bf16_t, PCB_CODE_INT8>(a, pl, stream);
    return a.code == PCB_CODE_E4M3 ? launch<float, PCB_CODE_E4M3>(a, pl, stream) : launch<float, PCB_CODE_INT8>(a, pl, stream);
}
