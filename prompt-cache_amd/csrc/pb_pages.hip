// The paged 8-bit cache beside its attention: a step's tables (pcb_page_tables), rows into pages and back (pcb_pages_append, pcb_pages_read).
//
// pcb_page_tables: every workgroup scans all sequences (a thread a sequence, in chunks of the workgroup) and knows each chunk's prefix sums; the flat rows,
// tiles and pages of a chunk are then shared out among the workgroups, each found by a search in the chunk's sums in LDS.  A step's tables are bound by the
// latency of the loads and of three scans one after the other, so a batch of one chunk and few rows is one workgroup.  Measured: 64 sequences of one token 6.6 us, 517 sequences
// and 95 700 rows 11.0.  Where the new lengths take the old ones' place there is one workgroup for all rows: 64 sequences and 13 900 rows 22 us, 517 and 99 300 141 (8 apart).
//
// pcb_pages_append / pcb_pages_read: a wave takes the rows of one page (reading: 4 to 32 rows, of any pages) of one head, keys or values, by itself: no LDS, no barrier, and
// the maximum of a page is a wave's reduction.  Both are bound by memory: rows in and codes out, each once.  Measured: 19 325 rows of 8 heads of 128 in and out again, 238 MB,
// 33.8 + 28.0 us = 3.8 TB/s; 8 247 rows of 32 heads out, 203 MB, 44.8 us = 4.5 TB/s (a copy reaches 4.9; into the same buffers again and again, which the last-level cache holds in
// part, 32.5).
#include "pb_pages.h"

namespace {
using namespace pcb;

// ---- tables -------------------------------------------------------------------------------------------------------------------------------
// K inclusive sums over the workgroup's threads; `all`: the whole sums.  One barrier: `part` belongs to one call of a chunk
template <int NT, int K, typename T>
__device__ __forceinline__ void block_scan(T (&v)[K], T (*part)[NT / 64], int tid, T (&all)[K]) {
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = wave_scan(v[k]);
        if (lane == 63) part[k][wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        all[k] = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            if (w == wave) v[k] += all[k];
            all[k] += part[k][w];
        }
    }
}
// the first thread whose sum is above x
template <int NT>
__device__ __forceinline__ int find(const int* sums, int x) {
    int lo = 0, hi = NT - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] > x)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}
__device__ __forceinline__ int ring_at(int64_t i, int cap) { return (int)(i % cap); }

template <int NT>
__global__ __launch_bounds__(NT) void page_tables_kernel(pcb_page_tables_args a, int ps) {
    __shared__ int64_t part64[1][NT / 64];
    __shared__ int part_need[1][NT / 64], part[5][NT / 64];
    __shared__ int stop_s[NT], take_s[NT], back_s[NT], tile_s[NT];    // inclusive sums over the chunk: rows, pages taken, pages given back, tiles
    __shared__ int cached_s[NT], have_s[NT], keep_s[NT], count_s[NT]; // count: rows of a granted sequence, -1 where not granted
    __shared__ int last;
    const int tid = threadIdx.x, P = 1 << ps, gsz = gridDim.x, wg = blockIdx.x;
    const int cap = a.ring ? a.ring_cap : 1;
    int head = a.ring ? a.ring_state[0] % cap : 0, free_pages = a.ring ? a.ring_state[1] : 0;
    head = head < 0 ? head + cap : head;                              // (a state that no call wrote stays inside the ring all the same)
    free_pages = free_pages < 0 ? 0 : free_pages > cap ? cap : free_pages;
    int64_t rows0 = 0;                                                // totals of the chunks before this one
    int need0 = 0, take0 = 0, back0 = 0, tile0 = 0, refused = 0, given = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += NT) {
        const int s = s0 + tid;
        const bool live = s < a.n_seqs;
        const int cached = live && a.cached[s] > 0 ? a.cached[s] : 0;
        const int brings = live ? a.brings[s] : 0;
        const bool over = brings < 0;
        const int count = over ? 0 : brings;
        const int have = (int)(((int64_t)cached + P - 1) >> ps);
        const int64_t total = ((int64_t)cached + count + P - 1) >> ps;
        int64_t rows_sum[1] = {(int64_t)count}, rows_whole[1];
        block_scan<NT>(rows_sum, part64, tid, rows_whole);
        const int64_t rows_all = rows_whole[0], stop = rows0 + rows_sum[0];
        const bool fits = total <= a.max_pages && stop <= a.n_rows;
        const int need = a.ring && live && !over && fits ? (int)total - have : 0;
        int need_sum[1] = {need}, need_all[1];
        block_scan<NT>(need_sum, part_need, tid, need_all);
        const bool granted = live && !over && fits && (need == 0 || need0 + need_sum[0] <= free_pages);
        int keep = over && a.keep ? a.keep[s] : 0;
        keep = keep < 0 ? 0 : keep;
        const int back = a.ring && over && have <= a.max_pages && have > keep ? have - keep : 0;
        const int tiles = granted ? (int)(((int64_t)count + a.tile_rows - 1) / a.tile_rows) : 0;
        int sums[5] = {granted ? need : 0, back, tiles, live && !over && !granted ? 1 : 0, granted ? count : 0}, whole[5];
        block_scan<NT>(sums, part, tid, whole);
        const int take_all = whole[0], back_all = whole[1], tile_all = whole[2];
        take_s[tid] = sums[0], back_s[tid] = sums[1], tile_s[tid] = sums[2];
        refused += whole[3], given += whole[4];
        stop_s[tid] = (int)(stop - rows0 > a.n_rows ? (int64_t)a.n_rows + 1 : stop - rows0);   // (rows behind n_rows are nobody's)
        cached_s[tid] = cached, have_s[tid] = have, keep_s[tid] = keep, count_s[tid] = granted ? count : -1;
        if (wg == 0) {
            if (live) {
                if (a.kv_len) a.kv_len[s] = over ? 0 : granted ? cached + count : cached;
                if (a.row_start) {
                    const int64_t first = stop - count;
                    a.row_start[s] = (int)(first > 0x7fffffff ? 0x7fffffff : first);
                    if (s == a.n_seqs - 1) a.row_start[a.n_seqs] = (int)(stop > 0x7fffffff ? 0x7fffffff : stop);
                }
            }
        }
        __syncthreads();
        const int at0 = wg * NT + tid, step = gsz * NT;
        // the granted sequences' new pages, and the places of those that come back
        for (int i = at0; i < take_all; i += step) {
            const int t = find<NT>(take_s, i), j = i - (t ? take_s[t - 1] : 0);
            a.table[(int64_t)(s0 + t) * a.ld_table + have_s[t] + j] = a.ring[ring_at((int64_t)head + take0 + i, cap)];
        }
        for (int i = at0; i < back_all; i += step) {
            const int t = find<NT>(back_s, i), j = i - (t ? back_s[t - 1] : 0);
            a.ring[ring_at((int64_t)head + free_pages + back0 + i, cap)] = a.table[(int64_t)(s0 + t) * a.ld_table + keep_s[t] + j];
        }
        const int n_here = rows_all > a.n_rows ? a.n_rows : (int)rows_all;
        for (int i = at0; i < n_here; i += step) {
            const int64_t r = rows0 + i;
            if (r >= a.n_rows) break;
            const int t = find<NT>(stop_s, i), k = i - (t ? stop_s[t - 1] : 0);
            const int64_t pos = (int64_t)cached_s[t] + k;
            int64_t slot = -1;
            if (count_s[t] >= 0) {
                const int q = (int)(pos >> ps);
                const int before = t ? take_s[t - 1] : 0;
                const int page = a.ring && q >= have_s[t] ? a.ring[ring_at((int64_t)head + take0 + before + q - have_s[t], cap)]
                                                          : a.table[(int64_t)(s0 + t) * a.ld_table + q];
                if (page >= 0) slot = (int64_t)page * P + (pos & (P - 1));
            }
            if (a.row_seq) a.row_seq[r] = s0 + t;
            if (a.row_pos) a.row_pos[r] = (int)(pos > 0x7fffffff ? 0x7fffffff : pos);
            a.row_slot[r] = slot;
        }
        if (a.tiles)
            for (int i = at0; i < tile_all; i += step) {
                const int t = find<NT>(tile_s, i), off = (i - (t ? tile_s[t - 1] : 0)) * a.tile_rows;
                const int left = count_s[t] - off;
                int4 rec;
                rec.x = s0 + t, rec.y = cached_s[t] + off, rec.z = left < a.tile_rows ? left : a.tile_rows;
                rec.w = (int)(rows0 + (t ? stop_s[t - 1] : 0)) + off;
                if (tile0 + i < a.n_tiles) reinterpret_cast<int4*>(a.tiles)[tile0 + i] = rec;
            }
        rows0 += rows_all, need0 += need_all[0], take0 += take_all, back0 += back_all, tile0 += tile_all;
        __syncthreads();
    }
    for (int64_t r = rows0 + wg * NT + tid; r < a.n_rows; r += gsz * NT) {
        if (a.row_seq) a.row_seq[r] = -1;
        if (a.row_pos) a.row_pos[r] = -1;
        a.row_slot[r] = -1;
    }
    if (a.tiles)
        for (int64_t t = (int64_t)tile0 + wg * NT + tid; t < a.n_tiles; t += gsz * NT) reinterpret_cast<int4*>(a.tiles)[t] = int4{-1, 0, 0, 0};
    if (wg == 0 && tid == 0 && a.status) a.status[0] = refused, a.status[1] = given;
    if (!a.ring) return;
    // ring_out may be ring_state: it is written by the workgroup that arrives last, when all have read it
    __syncthreads();
    if (tid == 0) {
        last = gsz == 1 || atomicAdd(&a.ring_out[2], 1) == gsz - 1;
        if (last) {
            a.ring_out[0] = ring_at((int64_t)head + take0, cap);
            a.ring_out[1] = free_pages - take0 + back0;
            a.ring_out[2] = 0, a.ring_out[3] = 0;
        }
    }
}

// A wave a sequence; one that is over looks at the others, a lane each: pages are equal up to some place and nowhere behind it, so the place is found by halving.
__global__ __launch_bounds__(256) void pages_kept_kernel(int n_seqs, const int32_t* cached, const int32_t* brings, const int32_t* table, int64_t ld_table, int max_pages, int ps, int32_t* keep) {
    const int lane = threadIdx.x & 63, s = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (s >= n_seqs) return;
    auto pages_of = [&](int t) { return (int)min(((int64_t)max(cached[t], 0) + (1 << ps) - 1) >> ps, (int64_t)max_pages); };
    int most = 0;
    if (brings[s] < 0) {
        const int32_t* mine = table + (int64_t)s * ld_table;
        const int have = pages_of(s);
        for (int t = lane; t < n_seqs && have > 0; t += 64) {
            if (t == s || (brings[t] < 0 && t > s)) continue;
            const int32_t* other = table + (int64_t)t * ld_table;
            int lo = most, hi = min(have, pages_of(t));               // lo pages are equal, or the other way to as many has been found
            while (lo < hi) {
                const int mid = lo + (hi - lo + 1) / 2;
                if (mine[mid - 1] == other[mid - 1])
                    lo = mid;
                else
                    hi = mid - 1;
            }
            most = lo;
        }
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) most = max(most, __shfl_xor(most, x, 64));
    }
    if (lane == 0) keep[s] = most;
}

// ---- rows into pages ------------------------------------------------------------------------------------------------------------------------
// sixteen bytes of a row, CE elements
template <typename E>
struct Piece {
    static constexpr int CE = 16 / sizeof(E);
    u32x4 w;
    __device__ __forceinline__ float at(int e) const {
        if constexpr (sizeof(E) == 2)
            return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        else
            return __uint_as_float(w[e]);
    }
};
// the largest magnitude's bits among what `m` holds (bf16: pairs) and a piece: numbers order as their bits do, and what is no finite number comes out above them
__device__ __forceinline__ uint32_t larger(uint32_t m, const Piece<bf16_t>& p) {
    typedef uint16_t u2 __attribute__((ext_vector_type(2)));
    u2 r = __builtin_bit_cast(u2, m);
#pragma unroll
    for (int q = 0; q < 4; ++q) r = __builtin_elementwise_max(r, __builtin_bit_cast(u2, p.w[q] & 0x7fff7fffu));
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t larger(uint32_t m, const Piece<float>& p) {
#pragma unroll
    for (int q = 0; q < 4; ++q) m = max(m, p.w[q] & 0x7fffffffu);
    return m;
}
template <typename E>
__device__ __forceinline__ float largest(uint32_t m) { return __uint_as_float(sizeof(E) == 2 ? max(m & 0xffff0000u, m << 16) : m); }
__device__ __forceinline__ float size_of(float x) { return __builtin_fabsf(x) < __builtin_inff() ? __builtin_fabsf(x) : 0.0f; }

// four numbers within the codes' range, in units of 1 / inv, as codes.  int8: added to 1.5 2^23 a number is rounded to a whole one, which the last byte then is
template <int CODE>
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d, float inv) {
    if (CODE == PCB_CODE_E4M3) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, lo, true);
    }
    const float big = 12582912.0f;
    const uint32_t x = __builtin_amdgcn_perm(__float_as_uint(__builtin_fmaf(b, inv, big)), __float_as_uint(__builtin_fmaf(a, inv, big)), 0x0c0c0400u);
    const uint32_t y = __builtin_amdgcn_perm(__float_as_uint(__builtin_fmaf(d, inv, big)), __float_as_uint(__builtin_fmaf(c, inv, big)), 0x0c0c0400u);
    return x | y << 16;
}

// four codes anew, in units that are 1 / ratio times as large
template <int CODE>
__device__ __forceinline__ uint32_t again(uint32_t w, float ratio) {
    float o[4];
    from_codes<CODE>(w, o);
    return to_codes<CODE>(o[0] * ratio, o[1] * ratio, o[2] * ratio, o[3] * ratio);
}
// the bytes k .. 3 of a word
__device__ __forceinline__ uint32_t from_byte(int k) { return k >= 4 ? 0u : k <= 0 ? 0xffffffffu : 0xffffffffu << (8 * k); }

struct RowsView {
    const int64_t* slot;
    int n_rows, ps;
    int64_t slots;                                                    // of the whole pool
    __device__ __forceinline__ int64_t at(int64_t r) const {
        if (r < 0 || r >= n_rows) return -1;
        const int64_t s = slot[r];
        return s >= 0 && s < slots ? s : -1;
    }
};

// One wave: the rows r0 .. r0 + n - 1 (n <= P), all of one page, their first slot s0, their smallest place off_min; `even`: their slots follow one another.
//
// A lane takes sixteen rows, those whose places share a multiple of 16, and sixteen bytes of each: the maximum, a key row's codes and a value column's sixteen codes (one
// store) all come out of the same registers, and a page of 64 rows of 128 bf16 elements is one such load for the wave, read once.  (Rows first for the maximum, then again for
// the codes, value columns a row a lane at a time: 55 us for 19 325 rows of 8 heads.)  Larger pages are read twice, the second time as far as the caches held them: 9 600 rows of
// 8 x 128 in fp32 54 us = 1.8 TB/s, in pages of 128 93 = 1.1; bf16 in pages of 128 1.9, of 16, which leave lanes idle, 2.5, of 32 3.6, of 64 4.1.
template <typename E, int CODE, bool PAST, bool VALUES>
__device__ void append_run(const pcb_pages_rows_args& a, const RowsView& v, int64_t r0, int n, int64_t s0, int off_min, bool even, int h, int lane) {
    constexpr int CE = Piece<E>::CE;
    const int P = 1 << v.ps, dim = a.dim, cpr = dim / CE;             // pieces of a row
    const int64_t page = s0 >> v.ps;
    const int64_t ld = VALUES ? a.ldv : a.ldk;
    const E* src = (const E*)(VALUES ? a.v : a.k) + (int64_t)h * (VALUES ? a.v_head_stride : a.k_head_stride) + r0 * ld;
    float* scale = (VALUES ? a.vscale : a.kscale) + page * a.Hkv + h;
    uint8_t* codes = (uint8_t*)(VALUES ? a.vcodes : a.kcodes) + (page * a.Hkv + h) * (int64_t)P * dim;
    const float was = off_min > 0 ? *scale : 0.0f;                    // (asked for beside the rows)
    const int off0 = even ? (int)(s0 & (P - 1)) : 0, g0 = off0 >> 4;  // (rows in another order: sixteen as they come)
    const int tasks = (((off0 + n - 1) >> 4) - g0 + 1) * cpr;
    Piece<E> x[16];
    int f = 0, c = 0;                                                 // the lane's rows f .. f + 15, of which those in 0 .. n - 1 exist (the others repeat one), and its piece
    auto load = [&](int i) {
        const int grp = i / cpr;
        f = 16 * (g0 + grp) - off0, c = i - grp * cpr;
        const E* p = src + c * CE;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const u32x4* q = reinterpret_cast<const u32x4*>(p + min(max(f + k, 0), n - 1) * ld);
            x[k].w = PAST ? __builtin_nontemporal_load(q) : *q;
        }
    };
    uint32_t mb = 0;
    for (int i = lane; i < tasks; i += 64) {
        load(i);
#pragma unroll
        for (int k = 0; k < 16; ++k) mb = larger(mb, x[k]);
    }
    float m = wave_max(largest<E>(mb));                               // (as numbers: a NaN among them is passed over ..)
    const bool odd = __any(!(largest<E>(mb) <= code_top<CODE>() * 1099511627776.0f));   // .. but seen here; as are infinities, and numbers beyond the largest scale's range
    if (odd) {
        m = 0.0f;
        for (int i = lane; i < n * cpr; i += 64) {
            Piece<E> y;
            y.w = *reinterpret_cast<const u32x4*>(src + i / cpr * ld + i % cpr * CE);
#pragma unroll
            for (int e = 0; e < CE; ++e) m = fmaxf(m, size_of(y.at(e)));
        }
        m = wave_max(m);
    }
    float s = scale_for<CODE>(m);
    if (was >= s) {
        s = was;
    } else if (off_min > 0) {
        // the codes in front of the first new row, in the new units.  (An old scale of a page that this library wrote is a power of two.)
        const float ratio = was * inv_pow2(s);
        if (!VALUES) {
            uint32_t* w = (uint32_t*)codes;
            for (int i = lane; i < off_min * dim / 4; i += 64) w[i] = again<CODE>(w[i], ratio);
        } else {
            const int words = (off_min + 3) / 4;
            for (int i = lane; i < words * dim; i += 64) {
                const int d = i / words, k = i - d * words;
                uint32_t* w = (uint32_t*)(codes + (int64_t)d * P) + k;
                const uint32_t old = *w, now = again<CODE>(old, ratio), keep = from_byte(off_min - 4 * k);
                *w = (now & ~keep) | (old & keep);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // (other lanes take up the rest of these words)
        }
    }
    if (lane == 0) *scale = s;
    const float inv = inv_pow2(s);
    if (odd || !even) {                                               // element by element
        for (int i = lane; i < n * dim; i += 64) {
            const int r = i / dim, d = i - r * dim, off = (int)(v.at(r0 + r) & (P - 1));
            const uint8_t code = (uint8_t)to_codes<CODE>(to_f32(src[r * ld + d]) * inv, 0.f, 0.f, 0.f);
            codes[VALUES ? (int64_t)d * P + off : (int64_t)off * dim + d] = code;
        }
        return;
    }
    for (int i = lane; i < tasks; i += 64) {
        if (tasks > 64) load(i);
        const int lo = max(0, -f), hi = min(16, n - f);               // the lane's rows that exist
        if (!VALUES) {
            uint8_t* dst = codes + (int64_t)(off0 + f) * dim + c * CE;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                uint32_t w[CE / 4];
#pragma unroll
                for (int q = 0; q < CE / 4; ++q) w[q] = codes_of<CODE>(x[k].at(4 * q), x[k].at(4 * q + 1), x[k].at(4 * q + 2), x[k].at(4 * q + 3), inv);
                if (k < lo || k >= hi) continue;
                if constexpr (CE == 8)
                    *reinterpret_cast<u32x2*>(dst + k * dim) = u32x2{w[0], w[1]};
                else
                    *reinterpret_cast<uint32_t*>(dst + k * dim) = w[0];
            }
            continue;
        }
        u32x4* dst = reinterpret_cast<u32x4*>(codes + (int64_t)(c * CE) * P + off0 + f);
        const int step = P / 16;
        u32x4 keep;                                                   // what of the columns' pieces stays
#pragma unroll
        for (int q = 0; q < 4; ++q) keep[q] = ~from_byte(lo - 4 * q) | from_byte(hi - 4 * q);
        const bool some = lo > 0 || hi < 16;
#pragma unroll
        for (int e = 0; e < CE; ++e) {
            u32x4 w;
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = codes_of<CODE>(x[4 * q].at(e), x[4 * q + 1].at(e), x[4 * q + 2].at(e), x[4 * q + 3].at(e), inv);
            if (some) w = (w & ~keep) | (dst[e * step] & keep);
            dst[e * step] = w;
        }
    }
}

// blockIdx.y: keys or values.  A wave looks at `win` rows of one head and takes the runs that start there.
template <typename E, int CODE, bool PAST>
__global__ __launch_bounds__(256) void pages_append_kernel(pcb_pages_rows_args a, RowsView v, int win) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int h = (int)(unit % a.Hkv);
    const int64_t w0 = unit / a.Hkv * win;
    if (w0 >= a.n_rows) return;
    const int P = 1 << v.ps;
    const int64_t mine = lane < win ? v.at(w0 + lane) : -1;
    const int64_t prev = lane < win ? v.at(w0 + lane - 1) : -1;
    uint64_t starts = __ballot(mine >= 0 && (prev < 0 || prev >> v.ps != mine >> v.ps));
    while (starts) {
        const int i = __builtin_ctzll(starts);
        starts &= starts - 1;
        const int64_t r0 = w0 + i, s0 = __shfl(mine, i, 64), page = s0 >> v.ps;
        // how far the run goes, its smallest place and whether its slots follow one another (P <= 128: two looks)
        int n = 0, off_min = P;
        bool even = true, open = true;
        for (int part = 0; part < P && open; part += 64) {
            const int64_t s = part + lane < P ? v.at(r0 + part + lane) : -1;
            const uint64_t in = __ballot(s >= 0 && s >> v.ps == page);
            const int k = ~in ? __builtin_ctzll(~in) : 64;
            open = k == 64;
            n += k;
            int o = lane < k ? (int)(s & (P - 1)) : P;
#pragma unroll
            for (int x = 32; x > 0; x >>= 1) o = min(o, __shfl_xor(o, x, 64));
            off_min = min(off_min, o);
            if (__ballot(lane < k && s != s0 + part + lane)) even = false;
        }
        if (blockIdx.y == 0)
            append_run<E, CODE, PAST, false>(a, v, r0, n, s0, off_min, even, h, lane);
        else
            append_run<E, CODE, PAST, true>(a, v, r0, n, s0, off_min, even, h, lane);
    }
}

// ---- rows out of pages ------------------------------------------------------------------------------------------------------------------------
// eight neighbouring elements of a row; PAST: past the caches
template <bool PAST>
__device__ __forceinline__ void put16(void* p, u32x4 w) {
    if (PAST)
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
    else
        *reinterpret_cast<u32x4*>(p) = w;
}
template <bool PAST>
__device__ __forceinline__ void put8(bf16_t* p, const float (&o)[8]) {
    put16<PAST>(p, u32x4{bf16_pair(o[0], o[1]), bf16_pair(o[2], o[3]), bf16_pair(o[4], o[5]), bf16_pair(o[6], o[7])});
}
template <bool PAST>
__device__ __forceinline__ void put8(float* p, const float (&o)[8]) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
        put16<PAST>(p + 4 * q, u32x4{__float_as_uint(o[4 * q]), __float_as_uint(o[4 * q + 1]), __float_as_uint(o[4 * q + 2]), __float_as_uint(o[4 * q + 3])});
}

// A wave takes `win` rows of one head, keys or values.  Keys: a lane eight codes of a row.  Values: rows whose slots follow one another within sixteen are a group, and a lane takes
// eight columns of one, sixteen codes each, and stores eight elements a row.
template <typename E, int CODE, bool PAST>
__global__ __launch_bounds__(256) void pages_read_kernel(pcb_pages_rows_args a, RowsView v, int win) {
    const int lane = threadIdx.x & 63, dim = a.dim, P = 1 << v.ps, cpr = dim / 8;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int h = (int)(unit % a.Hkv);
    const int64_t w0 = unit / a.Hkv * win;
    if (w0 >= a.n_rows) return;
    const int64_t mine = lane < win ? v.at(w0 + lane) : -1;
    if (blockIdx.y == 0) {
        for (int i = lane; i - lane < win * cpr; i += 64) {
            const int r = i / cpr, c = i - r * cpr;
            const int64_t s = __shfl(mine, r < win ? r : 0, 64);
            if (r >= win || s < 0) continue;
            const int64_t page = s >> v.ps;
            const u32x2 w = *reinterpret_cast<const u32x2*>((const uint8_t*)a.kcodes + ((page * a.Hkv + h) * P + (s & (P - 1))) * dim + c * 8);
            const float sc = a.kscale[page * a.Hkv + h];
            float o[8];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float x[4];
                from_codes<CODE>(w[q], x);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[4 * q + j] = x[j] * sc;
            }
            put8<PAST>((E*)a.k + (w0 + r) * a.ldk + (int64_t)h * a.k_head_stride + c * 8, o);
        }
        return;
    }
    const int64_t prev = __shfl_up(mine, 1, 64);
    const uint64_t there = __ballot(mine >= 0), starts = __ballot(mine >= 0 && (lane == 0 || prev < 0 || prev + 1 != mine || mine % 16 == 0));
    const int side = 64 / cpr, my = lane / cpr, c = lane - my * cpr, n_starts = __popcll(starts);   // groups side by side (cpr <= 32)
    for (int at = 0; at < n_starts; at += side) {
        uint64_t left = starts;
        for (int k = 0; k < at + my; ++k) left &= left - 1;           // (my group: the at + my'th)
        const bool mine_too = my < side && left != 0;
        const int i = mine_too ? __builtin_ctzll(left) : 0;
        const int64_t s0 = __shfl(mine, i, 64);
        if (!mine_too) continue;
        uint64_t stop = i < 63 ? ((starts | ~there) >> (i + 1)) : 0;
        const int n = min(stop ? __builtin_ctzll(stop) + 1 : 64 - i, win - i);
        const int64_t page = s0 >> v.ps;
        const int first = (int)(s0 & 15);
        const float sc = a.vscale[page * a.Hkv + h];
        const uint8_t* codes = (const uint8_t*)a.vcodes + (page * a.Hkv + h) * (int64_t)P * dim + (int64_t)(8 * c) * P + (s0 & (P - 1) & ~15);
        u32x4 w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = *reinterpret_cast<const u32x4*>(codes + e * P);
        E* dst = (E*)a.v + (w0 + i - first) * a.ldv + (int64_t)h * a.v_head_stride + 8 * c;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[8][4];
#pragma unroll
            for (int e = 0; e < 8; ++e) from_codes<CODE>(w[e][q], x[e]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 4 * q + j;
                if (k < first || k >= first + n) continue;
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = x[e][j] * sc;
                put8<PAST>(dst + k * a.ldv, o);
            }
        }
    }
}

int check_rows(const pcb_pages_rows_args* a, const char* who) {
    PCB_REQUIRE(a && a->struct_bytes == sizeof(pcb_pages_rows_args), PCB_ERR_ARG, "%s: struct size mismatch", who);
    PCB_REQUIRE((a->dtype == PCB_BF16 || a->dtype == PCB_F32) && (a->code == PCB_CODE_E4M3 || a->code == PCB_CODE_INT8), PCB_ERR_ARG, "%s: unknown dtype or code", who);
    PCB_REQUIRE(a->n_rows >= 0 && a->n_pages > 0 && pcb_page_size_ok(a->page_size) && a->Hkv > 0 && a->dim > 0 && a->dim <= 256 && a->dim % 16 == 0, PCB_ERR_ARG,
                "%s: bad sizes (pages of 16, 32, 64 or 128 tokens, heads of a multiple of 16 up to 256)", who);
    if (a->n_rows == 0) return PCB_OK;
    const int es = a->dtype == PCB_BF16 ? 8 : 4;
    PCB_REQUIRE(a->k && a->v && a->row_slot && a->kcodes && a->kscale && a->vcodes && a->vscale, PCB_ERR_ARG, "%s: null pointer", who);
    PCB_REQUIRE(((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->kcodes | (uintptr_t)a->vcodes) % 16 == 0 && (uintptr_t)a->row_slot % 8 == 0 && a->ldk % es == 0 &&
                    a->ldv % es == 0 && a->k_head_stride % es == 0 && a->v_head_stride % es == 0,
                PCB_ERR_ARG, "%s: rows, heads and codes start on 16 bytes", who);
    PCB_REQUIRE(((int64_t)a->n_rows + 15) / 16 * a->Hkv <= (int64_t)1 << 25, PCB_ERR_ARG, "%s: too many rows (n_rows * Hkv up to 2^29)", who);
    return PCB_OK;
}

}  // namespace

PCB_EXPORT int pcb_page_tables(const pcb_page_tables_args* a, void* stream) {
    PCB_REQUIRE(a && a->struct_bytes == sizeof(pcb_page_tables_args), PCB_ERR_ARG, "pcb_page_tables: struct size mismatch");
    PCB_REQUIRE(a->n_seqs > 0 && a->max_pages > 0 && a->ld_table >= a->max_pages && pcb_page_size_ok(a->page_size) && a->n_rows >= 0 && a->n_rows <= 1 << 30 &&
                    (int64_t)a->n_seqs * a->max_pages < 0x7fffffff && (int64_t)a->max_pages * a->page_size <= 0x7fffffff,
                PCB_ERR_ARG, "pcb_page_tables: bad sizes (pages of 16, 32, 64 or 128 tokens, positions of 31 bits, up to 2^30 rows)");
    PCB_REQUIRE(a->cached && a->brings && a->table && (a->row_slot || a->n_rows == 0), PCB_ERR_ARG, "pcb_page_tables: null pointer");
    PCB_REQUIRE(!a->ring || (a->ring_cap > 0 && a->ring_state && a->ring_out), PCB_ERR_ARG, "pcb_page_tables: a ring comes with its state, and a place for the new one");
    PCB_REQUIRE(!a->tiles || (a->tile_rows > 0 && (uintptr_t)a->tiles % 16 == 0 && a->n_tiles >= (int64_t)a->n_seqs + a->n_rows / a->tile_rows), PCB_ERR_ARG,
                "pcb_page_tables: tiles on 16 bytes, n_seqs + n_rows / tile_rows of them");
    pcb_page_tables_args b = *a;
    if (!b.tiles) b.tile_rows = 1, b.n_tiles = 0;
    // one workgroup while a chunk holds all sequences and four trips all rows; never more where kv_len is `cached`, which the others still read.
    const bool one = a->kv_len == a->cached || (a->n_seqs <= 1024 && a->n_rows <= 4096);
    int groups = one ? 1 : pcb_ceil_div(a->n_rows > a->n_seqs ? a->n_rows : a->n_seqs, 1024);
    if (groups > 128) groups = 128;
    if (groups < 1) groups = 1;
    const int ps = pcb_log2(a->page_size);
    if (a->n_seqs <= 256 && a->n_rows <= 1024)
        hipLaunchKernelGGL(page_tables_kernel<256>, dim3(groups), dim3(256), 0, (hipStream_t)stream, b, ps);
    else
        hipLaunchKernelGGL(page_tables_kernel<1024>, dim3(groups), dim3(1024), 0, (hipStream_t)stream, b, ps);
    return pcb_check_launch("page_tables_kernel");
}

PCB_EXPORT int pcb_pages_kept(int32_t n_seqs, const int32_t* cached, const int32_t* brings, const int32_t* table, int64_t ld_table, int32_t max_pages, int32_t page_size, int32_t* keep,
                              void* stream) {
    PCB_REQUIRE(n_seqs > 0 && max_pages > 0 && ld_table >= max_pages && pcb_page_size_ok(page_size) && (int64_t)n_seqs * max_pages < 0x7fffffff, PCB_ERR_ARG,
                "pcb_pages_kept: bad sizes (pages of 16, 32, 64 or 128 tokens)");
    PCB_REQUIRE(cached && brings && table && keep, PCB_ERR_ARG, "pcb_pages_kept: null pointer");
    hipLaunchKernelGGL(pages_kept_kernel, dim3(pcb_ceil_div(n_seqs, 4)), dim3(256), 0, (hipStream_t)stream, n_seqs, cached, brings, table, ld_table, max_pages, pcb_log2(page_size), keep);
    return pcb_check_launch("pages_kept_kernel");
}

#define PCB_PAGES_LAUNCH2(KERNEL, E, CODE, PAST, GRID, ...)                                                                        \
    do {                                                                                                                         \
        if (PAST)                                                                                                                \
            hipLaunchKernelGGL((KERNEL<E, CODE, true>), GRID, dim3(256), 0, (hipStream_t)stream, *a, __VA_ARGS__);               \
        else                                                                                                                     \
            hipLaunchKernelGGL((KERNEL<E, CODE, false>), GRID, dim3(256), 0, (hipStream_t)stream, *a, __VA_ARGS__);              \
    } while (0)
#define PCB_PAGES_LAUNCH(KERNEL, PAST, GRID, ...)                                                                                \
    do {                                                                                                                         \
        if (a->dtype == PCB_BF16 && a->code == PCB_CODE_E4M3)                                                                    \
            PCB_PAGES_LAUNCH2(KERNEL, pcb::bf16_t, PCB_CODE_E4M3, PAST, GRID, __VA_ARGS__);                                      \
        else if (a->dtype == PCB_BF16)                                                                                           \
            PCB_PAGES_LAUNCH2(KERNEL, pcb::bf16_t, PCB_CODE_INT8, PAST, GRID, __VA_ARGS__);                                      \
        else if (a->code == PCB_CODE_E4M3)                                                                                       \
            PCB_PAGES_LAUNCH2(KERNEL, float, PCB_CODE_E4M3, PAST, GRID, __VA_ARGS__);                                            \
        else                                                                                                                     \
            PCB_PAGES_LAUNCH2(KERNEL, float, PCB_CODE_INT8, PAST, GRID, __VA_ARGS__);                                            \
    } while (0)

// Rows that are more than the L2 caches hold (32 MB) go past them, in and out (us): 8 247 rows of 32 heads of 128 in bf16 read from the pool 47.5 -> 32.6, 19 325 of 8 heads
// appended and read back 67.9 -> 61.2 by the loads.  Fewer come out of the caches or stay there for whoever reads them next.  (The codes themselves past them: 67.9 -> 70.9.)
static bool past_caches(const pcb_pages_rows_args* a) {
    return (int64_t)a->n_rows * a->Hkv * a->dim * (a->dtype == PCB_BF16 ? 4 : 8) > (int64_t)32 << 20;
}
// .. but not the rows of an append whose pages are more than one load of a wave, which are read twice (19 325 rows of 8 heads of 128, fp32 68.2 -> 62.7, bf16 in pages of 128 65.3 -> 61.8;
// 6 000 of 8 x 256, fp32, pages of 128 116.2 -> 104.7)
static bool read_once(const pcb_pages_rows_args* a) { return a->page_size / 16 * a->dim / (a->dtype == PCB_BF16 ? 8 : 4) <= 64; }
// rows that a wave looks at: as many as leave the chip's 1024 SIMDs four waves each or more, keys' and values' together, at most 64
static int window(int n_rows, int Hkv, int least, int most) {
    int w = least;
    while (w < most && (int64_t)n_rows * Hkv * 2 / (2 * w) >= 4096) w *= 2;
    return w;
}

PCB_EXPORT int pcb_pages_append(const pcb_pages_rows_args* a, void* stream) {
    const int rc = check_rows(a, "pcb_pages_append");
    if (rc != PCB_OK || a->n_rows == 0) return rc;
    const RowsView v{a->row_slot, a->n_rows, pcb_log2(a->page_size), (int64_t)a->n_pages * a->page_size};
    const int win = window(a->n_rows, a->Hkv, 1, a->page_size < 64 ? 32 : 64);   // (rows of different requests side by side; prompts: a page or two start in a window)
    const int64_t waves = ((int64_t)a->n_rows + win - 1) / win * a->Hkv;
    const dim3 grid((unsigned)((waves + 3) / 4), 2);
    PCB_PAGES_LAUNCH(pages_append_kernel, past_caches(a) && read_once(a), grid, v, win);
    return pcb_check_launch("pages_append_kernel");
}

PCB_EXPORT int pcb_pages_read(const pcb_pages_rows_args* a, void* stream) {
    const int rc = check_rows(a, "pcb_pages_read");
    if (rc != PCB_OK || a->n_rows == 0) return rc;
    PCB_REQUIRE(((a->ldk != 0 && a->ldv != 0) || a->n_rows == 1) && ((a->k_head_stride != 0 && a->v_head_stride != 0) || a->Hkv == 1), PCB_ERR_ARG,
                "pcb_pages_read: results have places of their own");
    const RowsView v{a->row_slot, a->n_rows, pcb_log2(a->page_size), (int64_t)a->n_pages * a->page_size};
    const int win = window(a->n_rows, a->Hkv, 4, 32);
    const int64_t waves = ((int64_t)a->n_rows + win - 1) / win * a->Hkv;
    const dim3 grid((unsigned)((waves + 3) / 4), 2);
    PCB_PAGES_LAUNCH(pages_read_kernel, past_caches(a), grid, v, win);
    return pcb_check_launch("pages_read_kernel");
}
