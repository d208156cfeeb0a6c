// Pieces that the kernels of the paged 8-bit cache share: codes as numbers and back, page addresses, scales.
//
// A scale is a power of two, kept as the float it is: products with it are exact, so a code * scale has one value however it is computed, a page whose scale
// grows moves its e4m3 codes without rounding them again (but for those that become subnormal), and the reciprocal is an exponent's negation.  Against the
// scale that would use the whole range it costs up to one bit of int8's seven and nothing of e4m3's relative step.
#pragma once
#include "pb_common.h"

static inline bool pcb_page_size_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }
static inline int pcb_log2(int p) { return p == 16 ? 4 : p == 32 ? 5 : p == 64 ? 6 : 7; }

#ifdef __HIPCC__
namespace pcb {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float fp2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// inclusive sums over a wave of which all lanes are active: within rows of sixteen, then their last lanes' over the next rows (no LDS, 6 steps)
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t moved(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)moved<CTRL, ROWS>((int)v) | (uint64_t)(uint32_t)moved<CTRL, ROWS>((int)(v >> 32)) << 32);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v += moved<0x111, 0xf>(v);                                        // row_shr 1, 2, 4, 8
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);                                        // row_bcast 15, 31
    return v + moved<0x143, 0xc>(v);
}

constexpr int SCALE_EXP = 40;      // exponents of scales: -40 .. 40.  The softmax weights times two scales' quotient then stay far inside fp32

template <int CODE>
__device__ __forceinline__ constexpr float code_top() { return CODE == PCB_CODE_E4M3 ? 448.0f : 127.0f; }

// the smallest power of two s (within the exponents' range) with m <= top * s, m >= 0 and finite: top = 1.75 * 2^8 or 1.984375 * 2^6, so the exponent of m less
// 8 or 6, one more where m's mantissa is above top's
template <int CODE>
__device__ __forceinline__ float scale_for(float m) {
    const uint32_t b = __float_as_uint(m);
    int e = (int)(b >> 23) - 127 - (CODE == PCB_CODE_E4M3 ? 8 : 6);
    if ((b & 0x7fffffu) > (CODE == PCB_CODE_E4M3 ? 0x600000u : 0x7e0000u)) ++e;
    e = e < -SCALE_EXP ? -SCALE_EXP : e > SCALE_EXP ? SCALE_EXP : e;
    return __uint_as_float((uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ float inv_pow2(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }
__device__ __forceinline__ float exp_of(float s) { return (float)((int)(__float_as_uint(s) >> 23) - 127); }

// x in units of the scale -> within the codes' range; what is not a number: 0
template <int CODE>
__device__ __forceinline__ float into_range(float x) {
    const float c = __builtin_fminf(__builtin_fmaxf(x, -code_top<CODE>()), code_top<CODE>());
    return x == x ? c : 0.0f;
}
// four numbers in units of the scale as four codes, to the nearest, ties to even
template <int CODE>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    a = into_range<CODE>(a), b = into_range<CODE>(b), c = into_range<CODE>(c), d = into_range<CODE>(d);
    if (CODE == PCB_CODE_E4M3) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
    }
    const uint32_t w = (uint32_t)(int)__builtin_rintf(a) & 255u, x = (uint32_t)(int)__builtin_rintf(b) & 255u, y = (uint32_t)(int)__builtin_rintf(c) & 255u,
                   z = (uint32_t)(int)__builtin_rintf(d) & 255u;
    return w | x << 8 | y << 16 | z << 24;
}
// four codes as the numbers they are in units of the scale
template <int CODE>
__device__ __forceinline__ void from_codes(uint32_t w, float (&o)[4]) {
    if (CODE == PCB_CODE_E4M3) {
        const fp2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        o[0] = a[0], o[1] = a[1], o[2] = b[0], o[3] = b[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = (float)((int)(w << (24 - 8 * i)) >> 24);
    }
}
// eight codes as eight halves, exactly: e4m3 numbers and -128 .. 127 both are halves.  int8: the byte plus 128 under the exponent of 1024 is 1024 + 128 + code
template <int CODE>
__device__ __forceinline__ h8 half8(u32x2 w) {
    h2 p[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (CODE == PCB_CODE_E4M3) {
            p[2 * i] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false));
            p[2 * i + 1] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true));
        } else {
            const uint32_t u = w[i] ^ 0x80808080u;
            const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
            p[2 * i] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
            p[2 * i + 1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
        }
    }
    h8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[2 * i] = p[i][0], r[2 * i + 1] = p[i][1];
    return r;
}

}  // namespace pcb
#endif
