// Paged key / value memory: the page plan of a step, the write of new rows into the pages, the attention of one new row per
// request over its pages (see estts_page_plan, estts_page_write, estts_paged_attention in include/estts.h).
#include "common.h"

#include <type_traits>

namespace {

// x / d for x < 2^bits without a division, whose thirty instructions stand in the way of the first loads of a short call (one request of
// 100 rows 3.35 / 3.17 us, three of up to 2500, cut, 6.45 / 6.16): with s = ceil(log2 d) and
// m = ceil(2^(bits + s) / d), m d = 2^(bits + s) + e, e < d <= 2^s, so x m / 2^(bits + s) is less than 1/d above x / d.  bits + s <= 62.
struct Divisor {
    uint32_t m; int shift;
    __device__ __forceinline__ int of(uint32_t x) const { return (int)(((uint64_t)x * m) >> shift); }
};
Divisor divisor(uint32_t d, int bits) {
    int s = 0;
    while ((1ULL << s) < d) ++s;
    return {(uint32_t)(((1ULL << (bits + s)) + d - 1) / d), bits + s};
}

// x / page for any x below 2^32: pages are multiples of 16 rows
struct PageSize {
    Divisor sixteenths; int page;
    __device__ __forceinline__ int of(uint32_t x) const { return sixteenths.of(x >> 4); }
    __device__ __forceinline__ int holding(int rows) const { return of((uint32_t)rows + page - 1); }        // pages that so many rows take
};
PageSize page_size(int page) { return {divisor((uint32_t)page / 16, 28), page}; }

// ------------------------------------------------------------------------------------------------ page plan
// Whole-number work on a few kilobytes, bound by latency: a launch, the lengths, the scans, the stack or the table, the maps.  One
// workgroup scans the requests; the copies and the rows' places are then made by the same workgroup, or by a second launch
// of as many as it takes where there are more than PLAN_ROWS rows (one workgroup for all / two launches: 64 prompts of 2047 rows at most
// 67.6 / 6.7 us, 1000 requests that end, grow and arrive, 26000 rows, 67.5 / 9.9).  A step of 32 requests is one launch of 2.8 us, some 2 of
// which are the launch itself.
constexpr int PLAN_LDS = 4096;         // requests whose plan fits the LDS (four ints each); beyond that it lives in the caller's scratch

// A value from another lane, 0 where there is none: CTRL says which (row_shr 1, 2, 4, 8: that many lanes below in the row of 16; row_bcast 15, 31:
// the last lane of the row, of the half wave before), ROWS which rows of 16 take it.
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V from_lane(V v) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
    } else {
        const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
        const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
        return (V)(((unsigned long long)(unsigned)hi << 32) | lo);
    }
}

// inclusive prefix sum over the wave: no LDS, six additions (with shuffles, which go through the LDS, a plan of 32 requests took 4.5 us
// where it then took 3.7, one of 1000 13.9 and 12.7)
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
    v += from_lane<0x111, 0xf>(v);
    v += from_lane<0x112, 0xf>(v);
    v += from_lane<0x114, 0xf>(v);
    v += from_lane<0x118, 0xf>(v);
    v += from_lane<0x142, 0xa>(v);
    return v + from_lane<0x143, 0xc>(v);
}

// inclusive prefix sum over the workgroup's NT threads, and the total.  part: of this scan alone until every thread has passed another barrier.
template <int NT, typename V>
__device__ __forceinline__ V block_scan(V v, V* part, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    if (lane == 63) part[wave] = v;
    __syncthreads();
    V before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const V s = part[w];
        if (w < wave) before += s;
        total += s;
    }
    return v + before;
}

// first b with end[b] > x (ends do not decrease); B if there is none.  (Three looks at a time, so half as many waits, were no faster.)
__device__ __forceinline__ int first_past(const int* end, int B, int x) {
    int lo = 0, hi = B;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// What is known of each request after the scans.  Up to PLAN_LDS requests it is held in the LDS.
struct PagePlan {
    const int* row_end;        // end of its rows in a packed map (at most T); their number where the map is padded
    const int* back_end;       // pages given back up to and including it
    const int* page_end;       // pages granted up to and including it
    const int* len_of;         // its length, complemented where it gets no rows
    int height0, back, taken;  // the stack before the call, pages that come back to it, pages that are then taken off it
};
struct PageDivisors { PageSize page; Divisor row; };           // (row: of a padded map)
constexpr int PLAN_HEAD = 4;   // scratch of a plan in two launches: height0, back, taken, then the four arrays

// The copies that a plan asks for, in any order and by any thread: every source is as the call found it.  Place e of the stack with the
// given-back pages on it is free_pages[e] below height0, above it the page of an ended request; a row's page is in the table if the
// request held it already, else on the stack.
template <bool PADDED, bool RUNS>
__device__ __forceinline__ void carry_out(const estts_page_plan_args& p, const PageDivisors& by, const PagePlan& q, const int first, const int step) {
    auto given_back = [&](int g) {
        const int b = first_past(q.back_end, p.B, g);
        return p.block_table[b * p.ld_table + (g - (b ? q.back_end[b - 1] : 0))];
    };
    auto on_stack = [&](int e) { return e < q.height0 ? p.free_pages[e] : given_back(e - q.height0); };
    const int height = q.height0 + q.back;
    // rows, pages taken and pages given back one behind the other, so that threads without rows begin with the pages at once
    const int rows = (p.T + 63) & ~63, work = rows + q.taken;           // (whole waves of rows)
    for (int x = first; x < work; x += step) {
        if (x >= rows) {
            const int g = x - rows, b = first_past(q.page_end, p.B, g);
            const int i = g - (b ? q.page_end[b - 1] : 0);
            p.block_table[b * p.ld_table + by.page.holding(q.len_of[b]) + i] = on_stack(height - 1 - g);
        } else if (x < p.T) {
            const int b = PADDED ? by.row.of(x) : first_past(q.row_end, p.B, x);
            int slot = -1, pos = -1;
            const int len = b < p.B ? q.len_of[b] : -1;
            if (len >= 0) {
                const int i = PADDED ? x - b * p.R : x - (b ? q.row_end[b - 1] : 0);
                if (!PADDED || i < q.row_end[b]) {
                    pos = len + i;
                    const int j = by.page.of(pos), fresh = j - by.page.holding(len);
                    const int id = fresh < 0 ? p.block_table[b * p.ld_table + j] : on_stack(height - 1 - ((b ? q.page_end[b - 1] : 0) + fresh));
                    if (id >= 0 && id < p.n_pages) slot = id * p.page + (pos - j * p.page);
                }
            }
            p.slots[x] = slot;
            if (p.positions) p.positions[x] = pos;
        }
    }
    if (!RUNS || q.back <= 4 * step) {
        const int behind = first - (int)((unsigned)work % (unsigned)step);
#pragma unroll 1
        for (int g = behind < 0 ? behind + step : behind; g < q.back; g += step) p.free_pages[q.height0 + g] = given_back(g);
        return;
    }
    // Many pages for few threads: a run for each wave, in pieces of one request's pages (at most 64), four in flight; looking each page up
    // by itself takes a thread 0.8 us a page (100 of 1000 requests of up to 4096 rows end: 16.3 us, like this 12.5).  Only in the kernel of
    // 1024 threads: the longer code alone costs the others 0.1 to 0.4 us.
    const int lane = first & 63, waves = step >> 6, per = (q.back + 64 * waves - 1) / (64 * waves) * 64;
    int g = __builtin_amdgcn_readfirstlane(first >> 6) * per;
    const int last = min(g + per, q.back);
    if (g >= last) return;
    int b = first_past(q.back_end, p.B, g);
    while (g < last) {
        int id[4], at[4], n[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            at[k] = g;
            n[k] = 0;
            if (g >= last) continue;
            const int end = q.back_end[b], from = b ? q.back_end[b - 1] : 0;
            n[k] = min(min(end, last) - g, 64);
            if (lane < n[k]) id[k] = p.block_table[b * p.ld_table + (g - from) + lane];
            g += n[k];
            if (g < end || g >= last) continue;
            uint64_t hit;                           // the next request that gives any back (there is one: g < back)
            do {
                const int x = b + 1 + lane;
                hit = __ballot(x < p.B && q.back_end[min(x, p.B - 1)] > g);
                b += hit ? __builtin_ctzll(hit) + 1 : 64;
            } while (!hit);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane < n[k]) p.free_pages[q.height0 + at[k] + lane] = id[k];
    }
}

// The scans, by one workgroup; then the copies, unless they are left to page_copy_kernel (SPLIT; the plan goes to p.ws).
template <int NT, bool LDS, bool PADDED, bool SPLIT>
__global__ __launch_bounds__(NT) void page_plan_kernel(const estts_page_plan_args p, const PageDivisors by) {
    __shared__ int back_s[NT / 64], need_s[2][NT / 64];
    __shared__ long long rows_s[NT / 64];
    __shared__ int taken_s, refused_s;
    __shared__ int plan_s[!LDS ? 1 : SPLIT ? PLAN_LDS : 4 * PLAN_LDS];
    const int tid = threadIdx.x;
    const int cap = p.P * p.page;
    const long pitch = LDS && !SPLIT ? PLAN_LDS : p.B;
    int* const plan = LDS && !SPLIT ? plan_s : p.ws + PLAN_HEAD;
    int *const row_end = plan, *const back_end = plan + pitch, *const page_end = plan + 2 * pitch, *const len_of = plan + 3 * pitch;
    int* const mark_of = LDS && SPLIT ? plan_s : len_of;        // (what a thread reads again itself)

    const int height0 = min(max(p.n_free[0], 0), p.n_pages);
    if (tid == 0) taken_s = refused_s = 0;
    // rows before each request; pages of the requests that ended (two scans a turn: the barrier of each lies between two uses of the other's sums)
    int back = 0;
    long long rows_before = 0;
    for (int b0 = 0; b0 < p.B; b0 += NT) {
        const int b = b0 + tid;
        const int n = b < p.B ? p.n_new[b] : 0;
        const int len = b < p.B ? min(max(p.lengths[b], 0), cap) : 0;
        int back_total;
        const int upto = back + block_scan<NT>(n < 0 ? by.page.holding(len) : 0, back_s, back_total);
        long long rows_total = 0, rows_upto = 0;
        if constexpr (PADDED) { if (b0 + NT < p.B) __syncthreads(); }       // (for back_s)
        else rows_upto = rows_before + block_scan<NT>((long long)max(n, 0), rows_s, rows_total);
        if (b < p.B) {
            back_end[b] = upto;
            const bool inside = n <= 0 || (PADDED ? n <= p.R : rows_upto <= p.T);
            row_end[b] = PADDED ? max(n, 0) : (int)min(rows_upto, (long long)p.T);
            mark_of[b] = inside ? len : ~len;
        }
        back += back_total;
        rows_before += rows_total;
    }
    back = min(back, p.n_pages - height0);          // (more would be pages that are held twice)
    const int height = height0 + back;
    // grants
    int asked = 0;
    for (int b0 = 0, turn = 0; b0 < p.B; b0 += NT, turn ^= 1) {         // (two sets of sums in turn: one barrier lies between uses of the same)
        const int b = b0 + tid;
        const int n = b < p.B ? p.n_new[b] : 0;
        const int mark = b < p.B ? mark_of[b] : 0, len = mark < 0 ? ~mark : mark;
        const bool fits = b < p.B && n >= 0 && mark >= 0 && len + (long long)n <= cap;
        const int need = fits ? by.page.holding(len + n) - by.page.holding(len) : 0;
        int need_total;
        const int upto = asked + block_scan<NT>(need, need_s[turn], need_total);
        const bool granted = fits && (need == 0 || upto <= height);
        if (b < p.B) {
            page_end[b] = min(upto, height);        // (a request that is turned away ends no page below its own)
            len_of[b] = granted ? len : ~len;
            p.lengths_out[b] = n < 0 ? 0 : granted ? len + n : len;
            if (granted && need) atomicMax(&taken_s, upto);
            if (n >= 0 && !granted) atomicAdd(&refused_s, 1);
        }
        asked += need_total;
    }
    __syncthreads();
    const int taken = taken_s;
    if (tid == 0) {
        p.n_free_out[0] = height - taken;
        if (p.refused) p.refused[0] = refused_s;
    }
    if constexpr (SPLIT) {
        if (tid == 0) { p.ws[0] = height0; p.ws[1] = back; p.ws[2] = taken; }
    } else {
        carry_out<PADDED, NT == 1024>(p, by, {row_end, back_end, page_end, len_of, height0, back, taken}, tid, NT);
    }
}

template <bool LDS, bool PADDED>
__global__ __launch_bounds__(256) void page_copy_kernel(const estts_page_plan_args p, const PageDivisors by) {
    __shared__ __attribute__((aligned(16))) int plan_s[LDS ? 4 * PLAN_LDS : 4];
    const int* plan = p.ws + PLAN_HEAD;
    const int height0 = p.ws[0], back = p.ws[1], taken = p.ws[2];
    if (LDS) {
        // (four loads in flight: one at a time this was most of the launch)
#pragma unroll 4
        for (int x = threadIdx.x; x < p.B; x += 256) reinterpret_cast<int4*>(plan_s)[x] = reinterpret_cast<const int4*>(plan)[x];
        __syncthreads();
        plan = plan_s;
    }
    carry_out<PADDED, false>(p, by, {plan, plan + p.B, plan + 2 * (long)p.B, plan + 3 * (long)p.B, height0, back, taken}, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ------------------------------------------------------------------------------------------------ rows into the pages
// Every byte moves once: bound by memory.  A thread takes 16 bytes of a row of the pages, of K and of V; 2^lanes_log threads side by side
// share a row, `cols` workgroups next to each other the wider ones, so that rows are read and pages written in long runs.  STREAM:
// stores that are not kept in the caches (nt), which writes faster where they would not stay anyway: 8000 rows of 8 heads of 128, float32
// (131 MB) 28.4 / 21.2 us plain / streaming (6.2 TB/s), 16411 rows bfloat16 (179 MB) 37.4 / 35.7, 200000 rows of one head of 32 17.5 / 13.8;
// but 33 rows 2.1 / 2.4, and rows just written are read next.  Two or four rows to a thread: the same or up to 4 % slower.
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void page_write_kernel(const estts_page_write_args p, const int lanes_log, const int cols) {
    constexpr int VEC = 16 / (int)sizeof(T);
    typedef __attribute__((ext_vector_type(VEC))) T vec_t;
    const int chunk = blockIdx.x / cols, col = blockIdx.x - chunk * cols;
    const int c = ((col << lanes_log) + (threadIdx.x & ((1 << lanes_log) - 1))) * VEC;
    const long t = (long)chunk * (256 >> lanes_log) + (threadIdx.x >> lanes_log);
    if (c >= p.heads * p.depth || t >= p.T) return;
    const unsigned slot = (unsigned)p.slots[t], page = (unsigned)p.page;
    if (slot >= (unsigned)p.n_pages * page) return;         // (-1, too)
    const int h = c / p.depth;
    const long at = (long)(slot / page) * p.s_page + (long)h * p.s_head + (long)(slot % page) * p.s_row + (c - h * p.depth);
    const f32x4* ks = reinterpret_cast<const f32x4*>(p.k + t * p.ldk + c);
    const f32x4* vs = reinterpret_cast<const f32x4*>(p.v + t * p.ldv + c);
    f32x4 k[VEC / 4], v[VEC / 4];
#pragma unroll
    for (int x = 0; x < VEC / 4; ++x) { k[x] = ks[x]; v[x] = vs[x]; }
    vec_t kt, vt;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        kt[e] = (T)k[e >> 2][e & 3];
        vt[e] = (T)v[e >> 2][e & 3];
    }
    vec_t* ka = reinterpret_cast<vec_t*>(static_cast<T*>(p.k_cache) + at);
    vec_t* va = reinterpret_cast<vec_t*>(static_cast<T*>(p.v_cache) + at);
    if constexpr (STREAM) {
        __builtin_nontemporal_store(kt, ka);
        __builtin_nontemporal_store(vt, va);
    } else {
        *ka = kt;
        *va = vt;
    }
}

// ------------------------------------------------------------------------------------------------ attention of one new row
// With t = scale log2(e) q . k_j and M = max_j t_j:  ctx = sum_j 2^(t_j - M) v_j / sum_j 2^(t_j - M), computed in one pass over the rows with a
// running maximum.  What has to move is the keys and values themselves, a few operations per byte: the kernel is laid out so that the
// loads never wait for the arithmetic and the arithmetic stays off the LDS.
//
// A wave sweeps tiles of 16 (float32, depth 128) or 32 rows for up to 16 query heads that share a key head, on the matrix cores:
//   S^T (16 rows x 16 queries) = K Q^T      A = K: lane (i, g) holds row i, elements 8g .. 8g+7 of a step of 32 (float32: 4g .. 4g+3 of 16)
//   O^T (16 features x 16 queries) += V^T P^T   A = V^T: row r of the result is feature r * depth/16 + e in tile e (feature_of), so that lane i
//       loads consecutive features of a row for several tiles, and every load of 16 lanes takes whole lines of V
// The result layout D[4g + j][i] puts the weights of rows 4g + j into lane (i, g), which is where the second product wants them: of
// two 16-row halves (16-bit types: k slot 8g + 4 half + j is row 16 half + 4g + j) or as they are (float32: k slot g).  Nothing crosses
// lanes but the maximum.  16-bit values of V are interleaved from rows to features with one v_perm_b32 per two values.
// The matrix cores round nothing here that float32 would keep: float32 pages run through the float32 instructions; for 16-bit pages
// the queries and the weights are split into bfloat16 pieces (three, 24 bits) or float16 pieces (two, 22 bits, behind a power of two that
// puts the largest element of the query at 2^13 and the largest weight at 2^14), whose products with the pages' values are exact.
// Scores, maxima, sums and outputs are float32.
// What bounds it: memory where there are rows enough (5.9 to 6.4 TB/s from 130 MB on; a kernel that only reads and adds gets 6.2), else the chain
// launch, lengths and table, keys, scores, weights, values, exchange (3.2 us for one request of 100 rows) and some 0.6 to 1.1 us more for
// each further tile of a wave.

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// Waves of a workgroup: four; eight for whole requests on the vector ALU, whose arithmetic they spread (4 heads of 64, float32, four / eight: one
// request of 600 rows 5.5 / 5.1 us, of 1000 7.1 / 6.7, 64 ragged ones of 600 9.6 / 9.3, one of 100 3.3 / 3.4; on the matrix cores, 32 heads on 8 of
// 128, bfloat16, one of 1000 12.3 / 12.7, 128 ragged ones of 1000 56.2 / 58.3; cut, 61 ragged ones 89.4 / 90.3).
constexpr int ATT_WAVES = 4, FEW_WAVES = 8;
// query heads per key head up to which the vector ALU takes them (see paged_attention_few_kernel)
constexpr int few_queries(int esize) { return esize == 4 ? 2 : 1; }

// 16-row halves of a wave's tile
constexpr int tile_halves(int depth, int esize) { return depth * esize == 512 ? 1 : 2; }

// which feature lane (matrix row) r holds as its e-th: consecutive ones, 16 bytes of them at a time over the 16 lanes
template <int DH, int ESIZE>
__host__ __device__ constexpr int feature_of(int r, int e) {
    constexpr int NV = DH / 16, RUN = NV * ESIZE < 16 ? NV : 16 / ESIZE;
    return (e / RUN) * (16 * RUN) + r * RUN + e % RUN;
}

// Cache policy of the loads of V (the nt bit): not kept in the caches on the way.  Where the rows are more than the caches hold from one
// call to the next this reads faster, where they are not it costs what they would have held (see stream_rows).  Not for K, whose
// lines are read by two instructions.
constexpr int LOAD_STREAM = 2;

template <typename T> struct Kv16 { typedef bf16x8 Frag; static constexpr int PIECES = 1; };      // (float32: not used)
template <> struct Kv16<__bf16> {
    typedef bf16x8 Frag;
    static constexpr int PIECES = 3;
    static __device__ __forceinline__ f32x4 mfma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Kv16<_Float16> {
    typedef f16x8 Frag;
    static constexpr int PIECES = 2;
    static __device__ __forceinline__ f32x4 mfma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// x = sum of the pieces up to 2^-24 (bfloat16) or 2^-22 (float16) of x; two values to a conversion
template <typename T>
__device__ __forceinline__ void split_pieces(const float (&x)[8], typename Kv16<T>::Frag (&f)[Kv16<T>::PIECES]) {
    typedef __attribute__((ext_vector_type(2))) T pair_t;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        f32x2_t r = {x[e], x[e + 1]};
#pragma unroll
        for (int n = 0; n < Kv16<T>::PIECES; ++n) {
            const pair_t h = __builtin_convertvector(r, pair_t);
            f[n][e] = h[0];
            f[n][e + 1] = h[1];
            if (n + 1 < Kv16<T>::PIECES) r -= __builtin_convertvector(h, f32x2_t);
        }
    }
}

// 16 bytes (8, 4) at byte `lane_at` + `at` behind a base that is the same for the whole wave: the base and `at` stay in scalar registers
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t wave_rows(const char* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, bytes, 0x00027000);
}

__device__ __forceinline__ int request_rows(const estts_paged_attention_args& p, int b) {
    return min(min(max(p.lengths[b], 0), p.P * p.page), p.max_len);
}

// How the rows are dealt out.  SPLIT false: a workgroup has a whole request (and a key head's queries).  Else all rows of all requests,
// in units of UNIT, are one line that is cut into equal parts, so that long and short requests keep the chip equally busy and no part
// is last; the host knows no lengths, the parts follow from them on the GPU.  A part holds whole requests, the end of one that began in
// an earlier part and the beginning of one that goes on in a later part: two places of scratch a part, 2k and 2k + 1, hold the latter two.
// What the host works out of a call's arguments: the page size, query heads per key head, groups of them, and how to divide by kv_heads and target.
struct PagedCall { PageSize page; int group, n_group, target; Divisor kv_heads, by_target; };
struct PagedSegment { int b, begin, end, place; bool whole; };      // rows [begin, end) of request b; place: of the scratch, unless whole

template <int NT, int UNIT, bool SPLIT>
struct PagedPart {
    int k, b, off, left, at;                    // requests from b on, of b the units from off on, left units in all; at: place of unit off of b in the line
    int parts, total;                           // part k holds units [floor(k total / parts), floor((k + 1) total / parts)) of the line

    static __device__ __forceinline__ int units_of(int rows) { return max((rows + UNIT - 1) / UNIT, 1); }      // (a request without rows still gets its zeros)

    // that unit x of the line is in: floor(((x + 1) parts - 1) / total), in float64 (below 2^38 over below 2^30: a quotient that is no whole number
    // is 2^-30 away from the next)
    __device__ __forceinline__ int part_of(int x) const { return (int)(((x + 1.0) * parts - 1.0) / total); }

    __device__ __forceinline__ bool find(const estts_paged_attention_args& p, const PagedCall& c, int part) {
        int first = part, skip = 0;
        at = left = total = 0;
        parts = p.B;
        if constexpr (SPLIT) {
            __shared__ int scan_s[NT / 64], found_s[2];
            const int per = (p.B + NT - 1) / NT, b0 = threadIdx.x * per, b1 = min(b0 + per, p.B);
            int mine = 0;                       // (the sum over all is at most 2^30: the caller keeps B * max_len below 2^36)
            for (int x = b0; x < b1; ++x) mine += units_of(request_rows(p, x));
            const int upto = block_scan<NT>(mine, scan_s, total);
            parts = min(c.target, total);
            const int share = total < c.target ? 1 : c.by_target.of(total), extra = total - share * parts;     // (extra < target <= 256)
            at = part * share + c.by_target.of(part * extra);
            left = share + c.by_target.of((part + 1) * extra) - c.by_target.of(part * extra);
            if (part < parts && upto > at && upto - mine <= at) {
                int x = b0, before = upto - mine;
                for (; x < b1 - 1; ++x) {
                    const int n = units_of(request_rows(p, x));
                    if (before + n > at) break;
                    before += n;
                }
                found_s[0] = x;
                found_s[1] = at - before;
            }
            __syncthreads();
            first = found_s[0];
            skip = found_s[1];
        }
        k = part;
        b = __builtin_amdgcn_readfirstlane(first);
        off = __builtin_amdgcn_readfirstlane(skip);
        return part < parts;
    }

    // the next rows to do; items (of the first key head's workgroups): where the join finds request b
    __device__ __forceinline__ PagedSegment next(const estts_paged_attention_args& p, int2* items) {
        const int rows = __builtin_amdgcn_readfirstlane(request_rows(p, b));
        const int n = units_of(rows), take = SPLIT ? min(n - off, left) : n;
        const PagedSegment s = {b, off * UNIT, min(rows, (off + take) * UNIT), 2 * k + (off == 0), !SPLIT || take == n};
        if (SPLIT && off == 0 && items) items[b] = make_int2(k, take == n ? 1 : part_of(at + n - 1) - k + 1);
        left -= take;
        at += take;
        off = 0;
        ++b;
        return s;
    }
};

// scratch of a split call: per place and query head the unnormalised output (relative to its maximum), then (maximum, sum); per request
// (part it begins in, number of parts it lies in)
struct PagedScratch {
    float* out; float2* ml; int2* items;
    __host__ __device__ PagedScratch(void* ws, int target, int H, int depth) {
        out = static_cast<float*>(ws);
        ml = reinterpret_cast<float2*>(out + 2L * target * H * depth);
        items = reinterpret_cast<int2*>(ml + 2L * target * H);
    }
    static __host__ __device__ long bytes(int target, int H, int depth, int B) { return 2L * target * H * (depth + 2) * 4 + (long)B * 8; }
};

// A wave's walk over its tiles t = wave, wave + NW, ... of rows [begin, end): where the 16-row halves of a tile lie in the caches.  A half
// lies in one page (page sizes are multiples of 16), so that its place is one number for the whole wave; the lanes hold the places of
// the next 64 halves, the table entries of the 64 after them are on their way.
template <int HALVES, int NW>
struct PageWalk {
    static constexpr int TILE = 16 * HALVES, PER_BLOCK = 64 / HALVES;
    const int* table;
    long s_page, s_row;                                 // in bytes
    PageSize page;
    int n_pages, max_len, begin, wave, lane;
    int entry, next_entry, at_lo, at_hi;                // of this lane's half: its page, its byte offset (negative: no such page)
    long at[HALVES];                                    // of the tile last located
    bool ok[HALVES];

    __device__ __forceinline__ PageWalk(const estts_paged_attention_args& p, const PagedCall& c, int b, int begin_, int wave_, int esize)
        : table(p.block_table + b * p.ld_table), s_page(p.s_page * esize), s_row(p.s_row * esize), page(c.page), n_pages(p.n_pages),
          max_len(p.max_len), begin(begin_), wave(wave_), lane(threadIdx.x & 63) {
        entry = entry_of(0);
        next_entry = entry_of(1);
        place(0);
    }
    // first row of half lane % HALVES of tile number block * PER_BLOCK + lane / HALVES
    __device__ __forceinline__ int half_row(int block) const {
        return begin + ((block * PER_BLOCK + lane / HALVES) * NW + wave) * TILE + 16 * (lane % HALVES);
    }
    // (bounded by max_len, which the host knows, not by the length: the table and the lengths are read side by side)
    __device__ __forceinline__ int entry_of(int block) const { return table[page.of(min(half_row(block), max_len - 1))]; }
    __device__ __forceinline__ void place(int block) {
        const int r = half_row(block);
        const bool there = entry >= 0 && entry < n_pages && r < max_len;
        const long x = there ? entry * s_page + (long)(r - page.of(r) * page.page) * s_row : -1L;
        at_lo = (int)(x & 0xFFFFFFFFL);
        at_hi = (int)(x >> 32);
    }
    // go to tile number it of the wave, the one after the last or the last again
    __device__ __forceinline__ void locate(int it, bool next) {
        if (next && it % PER_BLOCK == 0) {
            entry = next_entry;
            place(it / PER_BLOCK);
            next_entry = entry_of(it / PER_BLOCK + 1);
        }
        const int k = it % PER_BLOCK;
#pragma unroll
        for (int s = 0; s < HALVES; ++s) {
            const int lo = __builtin_amdgcn_readlane(at_lo, k * HALVES + s), hi = __builtin_amdgcn_readlane(at_hi, k * HALVES + s);
            ok[s] = hi >= 0;
            at[s] = hi >= 0 ? (long)(((unsigned long)(unsigned)hi << 32) | (unsigned)lo) : 0;            // (row 0 of page 0 is always there)
        }
    }
};

// what a workgroup works on: a request or a part of the line (`part`), key head hk, query heads h0 .. h0 + heads - 1 (at most MAXQ)
template <int MAXQ>
struct PagedUnit {
    int part, hk, h0, heads;
    __device__ __forceinline__ PagedUnit(const estts_paged_attention_args& p, const PagedCall& c) {
        // query groups of one key head next to each other on one XCD (workgroups whose numbers agree mod 8), whose L2 then holds the rows
        int unit = blockIdx.x, q = 0;
        if (MAXQ > 2 && c.n_group > 1) {
            const int k = unit >> 3;
            q = k % c.n_group;
            unit = (k / c.n_group) * 8 + (unit & 7);
        }
        part = c.kv_heads.of(unit);
        hk = unit - part * p.kv_heads;
        heads = min(MAXQ, c.group - q * MAXQ);
        h0 = hk * c.group + q * MAXQ;
    }
};

// The rows of a tile that count, a bit for each: in range, in a page that exists, not masked.  A lane looks at one row (mask: of row
// lane % TILE), the wave holds the answer.
template <int HALVES>
__device__ __forceinline__ uint32_t rows_that_count(int r0, int end, const bool (&ok)[HALVES], float mask) {
    const int row = threadIdx.x % (16 * HALVES);
    const bool there = HALVES == 2 && row >= 16 ? ok[HALVES - 1] : ok[0];
    const uint64_t bits = __ballot(there && r0 + row < end && mask == 0.0f);
    return HALVES == 2 ? (uint32_t)bits : (uint32_t)bits & 0xFFFFu;
}

// The waves' shares (o_s, m_s, l_s in the LDS) meet; to ctx, or to the scratch where the segment is not a whole request.
template <int NW, int MAXQ, int DH>
__device__ __forceinline__ void join_waves(const estts_paged_attention_args& p, const PagedUnit<MAXQ>& u, const PagedSegment& seg, const PagedScratch& ws,
                                           const float (*o_s)[MAXQ][DH], const float (*m_s)[MAXQ], const float (*l_s)[MAXQ]) {
    for (int x = threadIdx.x; x < u.heads * DH; x += NW * 64) {
        const int h = x / DH, d = x % DH;
        float top = m_s[0][h];
#pragma unroll
        for (int v = 1; v < NW; ++v) top = fmaxf(top, m_s[v][h]);
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int v = 0; v < NW; ++v) {
            const float c = __builtin_amdgcn_exp2f(m_s[v][h] - base);
            sum = fmaf(l_s[v][h], c, sum);
            acc = fmaf(o_s[v][h][d], c, acc);
        }
        if (seg.whole) {
            p.ctx[seg.b * p.ldo + (long)(u.h0 + h) * DH + d] = sum == 0.0f ? 0.0f : acc / sum;
        } else {
            const long at = (long)seg.place * p.H + u.h0 + h;
            ws.out[at * DH + d] = acc;
            if (d == 0) ws.ml[at] = make_float2(top, sum);
        }
    }
}

// SPLIT: the rows are cut into c.target parts.  (A kernel for each: the code of the cutting alone, not run, cost a short request 0.4 to 0.7 us,
// one of 100 rows float32 4.2 / 3.6.)
template <typename T, int DH, bool MASK, bool STREAM, bool SPLIT, int NW>
__global__ __launch_bounds__(NW * 64, 2) void paged_attention_kernel(const estts_paged_attention_args p, const PagedCall c) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int HALVES = tile_halves(DH, sizeof(T));
    constexpr int TILE = 16 * HALVES;
    constexpr uint32_t ALL_ROWS = HALVES == 2 ? 0xFFFFFFFFu : 0xFFFFu;
    constexpr int NV = DH / 16;                         // features of a row of V per lane = tiles of 16 features
    constexpr int VB = NV * (int)sizeof(T) < 16 ? NV * (int)sizeof(T) : 16;     // bytes of one load of them
    __shared__ __attribute__((aligned(16))) float o_s[NW][16][DH];
    __shared__ float m_s[NW][16], l_s[NW][16];

    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedUnit<16> u(p, c);
    const int heads = u.heads, h0 = u.h0;
    const PagedScratch ws(p.ws, c.target, p.H, DH);
    PagedPart<NW * 64, TILE * NW, SPLIT> part;
    if (!part.find(p, c, u.part)) return;
    do {
        const PagedSegment seg = part.next(p, h0 == 0 && threadIdx.x == 0 ? ws.items : nullptr);
        const int b = seg.b, begin = seg.begin, end = seg.end;
        PageWalk<HALVES, NW> walk(p, c, b, begin, wave, sizeof(T));

        // ---- queries
        const float qs = p.scale * 1.4426950408889634f;
        const bool live = i < heads;
        const float* qp = p.q + b * p.ldq + (long)(h0 + (live ? i : 0)) * DH;
        constexpr int QV = DH / 4;                          // elements of the query per lane
        float qx[QV];
#pragma unroll
        for (int s = 0; s < QV / 4; ++s) {
            // float32: step s of 16 features, lane g has 4g .. 4g+3; else step s / 2 of 32 features, lane g has 8g .. 8g+7
            const float4 v = *reinterpret_cast<const float4*>(qp + (F32 ? 16 * s + 4 * g : 32 * (s >> 1) + 8 * g + 4 * (s & 1)));
            qx[4 * s] = live ? v.x * qs : 0.0f;
            qx[4 * s + 1] = live ? v.y * qs : 0.0f;
            qx[4 * s + 2] = live ? v.z * qs : 0.0f;
            qx[4 * s + 3] = live ? v.w * qs : 0.0f;
        }
        float unscale = 1.0f;                               // what the scores are multiplied with (float16: undoes the query's power of two)
        if constexpr (!F32 && Kv16<T>::PIECES == 2) {
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < QV; ++e) top = fmaxf(top, fabsf(qx[e]));
            top = fmaxf(top, lane_xor16(top));
            top = fmaxf(top, lane_xor32(top));
            const int ex = max((int)(__builtin_bit_cast(uint32_t, top) >> 23), 14);
            const float up = __builtin_bit_cast(float, (267 - ex) << 23);
            unscale = __builtin_bit_cast(float, (ex - 13) << 23);
#pragma unroll
            for (int e = 0; e < QV; ++e) qx[e] *= up;
        }
        [[maybe_unused]] typename Kv16<typename std::conditional<F32, __bf16, T>::type>::Frag qf[F32 ? 1 : DH / 32][Kv16<T>::PIECES];
        if constexpr (!F32) {
#pragma unroll
            for (int s = 0; s < DH / 32; ++s) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = qx[8 * s + e];
                split_pieces<T>(t, qf[s]);
            }
        }

        // ---- the wave's tiles
        const int n_tiles = (end - begin + TILE - 1) / TILE;
        const int n_mine = __builtin_amdgcn_readfirstlane(n_tiles > wave ? (n_tiles - wave + NW - 1) / NW : 0);
        const char* kbase = static_cast<const char*>(p.k_cache) + u.hk * p.s_head * (long)sizeof(T);
        const char* vbase = static_cast<const char*>(p.v_cache) + u.hk * p.s_head * (long)sizeof(T);
        const int row_bytes = (int)(p.s_row * (long)sizeof(T));

        // registers of a tile
        constexpr int KL = F32 ? DH / 16 : DH / 32;         // 16-byte loads of K per half and lane
        constexpr int VW = NV * (int)sizeof(T) / 4;         // dwords of V per row and lane
        i32x4 kr[HALVES][KL];
        int vr[HALVES][4][VW];
        [[maybe_unused]] float mk;                          // mask of row lane % TILE of the tile
        const int k_lane = i * row_bytes + 16 * g;
        const int v_lane = 4 * g * row_bytes + i * VB;
        int half_bytes = 15 * row_bytes + DH * (int)sizeof(T);         // (0 behind the last tile: such loads reach no memory)
        auto load_k = [&](int it) {
#pragma unroll
            for (int s = 0; s < HALVES; ++s) {
                const auto rows = wave_rows(kbase + walk.at[s], half_bytes);
#pragma unroll
                for (int x = 0; x < KL; ++x) kr[s][x] = __builtin_amdgcn_raw_buffer_load_b128(rows, k_lane + 64 * x, 0, 0);
            }
            if constexpr (MASK) mk = p.key_mask[b * p.mask_sb + min(begin + (it * NW + wave) * TILE + lane % TILE, end - 1) * p.mask_ss];
        };
        constexpr int POLICY = STREAM ? LOAD_STREAM : 0;
        auto load_v = [&]() {
#pragma unroll
            for (int s = 0; s < HALVES; ++s) {
                const auto rows = wave_rows(vbase + walk.at[s], half_bytes);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (VW >= 4) {
#pragma unroll
                        for (int x = 0; x < VW / 4; ++x) {
                            const i32x4 t = __builtin_amdgcn_raw_buffer_load_b128(rows, v_lane + 256 * x, j * row_bytes, POLICY);
                            vr[s][j][4 * x] = t[0]; vr[s][j][4 * x + 1] = t[1]; vr[s][j][4 * x + 2] = t[2]; vr[s][j][4 * x + 3] = t[3];
                        }
                    } else if constexpr (VW == 2) {
                        const i32x2 t = __builtin_amdgcn_raw_buffer_load_b64(rows, v_lane, j * row_bytes, POLICY);
                        vr[s][j][0] = t[0]; vr[s][j][VW - 1] = t[1];
                    } else {
                        vr[s][j][0] = __builtin_amdgcn_raw_buffer_load_b32(rows, v_lane, j * row_bytes, POLICY);
                    }
                }
            }
        };

        f32x4 o[NV];
#pragma unroll
        for (int e = 0; e < NV; ++e) o[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;                      // of query i; l: this lane's rows only
        constexpr float LIFT = std::is_same<T, _Float16>::value ? 14.0f : 0.0f;      // (the power of two on the weights)

        if (n_mine > 0) {
            walk.locate(0, false);
            load_k(0);
            load_v();
            bool ok_now[HALVES];
            for (int it = 0; it < n_mine; ++it) {
#pragma unroll
                for (int s = 0; s < HALVES; ++s) ok_now[s] = walk.ok[s];
                const int r0 = begin + (it * NW + wave) * TILE;
                // scores
                float sc[HALVES][4];
                if constexpr (F32) {
#pragma unroll
                    for (int s = 0; s < HALVES; ++s) {
                        f32x4 a0 = {0.0f, 0.0f, 0.0f, 0.0f}, a1 = a0;
#pragma unroll
                        for (int x = 0; x < KL; ++x) {
                            const f32x4 kf = __builtin_bit_cast(f32x4, kr[s][x]);
                            a0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[0], qx[4 * x], a0, 0, 0, 0);
                            a1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[1], qx[4 * x + 1], a1, 0, 0, 0);
                            a0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[2], qx[4 * x + 2], a0, 0, 0, 0);
                            a1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[3], qx[4 * x + 3], a1, 0, 0, 0);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[s][j] = a0[j] + a1[j];
                    }
                } else {
                    f32x4 acc[HALVES][Kv16<T>::PIECES];
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int n = 0; n < Kv16<T>::PIECES; ++n) acc[s][n] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int x = 0; x < KL; ++x)
#pragma unroll
                        for (int n = 0; n < Kv16<T>::PIECES; ++n)
#pragma unroll
                            for (int s = 0; s < HALVES; ++s)
                                acc[s][n] = Kv16<T>::mfma(__builtin_bit_cast(typename Kv16<T>::Frag, kr[s][x]), qf[x][n], acc[s][n]);
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float t = acc[s][Kv16<T>::PIECES - 1][j];
#pragma unroll
                            for (int n = Kv16<T>::PIECES - 2; n >= 0; --n) t += acc[s][n][j];
                            sc[s][j] = Kv16<T>::PIECES == 2 ? t * unscale : t;
                        }
                }
                // rows that count: in range, in a page that exists, not masked
                bool all_in = r0 + TILE <= end;
#pragma unroll
                for (int s = 0; s < HALVES; ++s) all_in = all_in && ok_now[s];
                uint32_t rows_in = 0;                       // a bit for each
                bool drop = !all_in;
                if (MASK || drop) {
                    rows_in = rows_that_count<HALVES>(r0, end, ok_now, MASK ? mk : 0.0f);
                    drop = rows_in != ALL_ROWS;
                }
                // the next tile's keys, into the registers just read (loads of nothing where there is none: the number of loads in flight
                // stays the same on every path, so that no wait is longer than it has to be)
                const int nx = min(it + 1, n_mine - 1);
                walk.locate(nx, nx != it);
                if (nx == it) half_bytes = 0;
                load_k(nx);
                if (drop) {
                    const uint32_t mine = rows_in >> (4 * g);
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const bool in = mine >> (16 * s + j) & 1;
                            sc[s][j] = in ? sc[s][j] : -INFINITY;
#pragma unroll
                            for (int x = 0; x < VW; ++x) vr[s][j][x] = in ? vr[s][j][x] : 0;       // (0 x NaN would be NaN)
                        }
                }
                // softmax step
                float top = sc[0][0];
#pragma unroll
                for (int s = 0; s < HALVES; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = fmaxf(top, sc[s][j]);
                top = fmaxf(top, lane_xor16(top));
                top = fmaxf(top, lane_xor32(top));
                if (__any(top > m)) {
                    const float m1 = fmaxf(m, top);
                    const float c = m1 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m1);
                    m = m1;
                    l *= c;
#pragma unroll
                    for (int e = 0; e < NV; ++e)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[e][j] *= c;
                }
                const float base = (m == -INFINITY ? 0.0f : m) - LIFT;
                float pw[8];
#pragma unroll
                for (int s = 0; s < HALVES; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        pw[4 * s + j] = __builtin_amdgcn_exp2f(sc[s][j] - base);
                        l += pw[4 * s + j];
                    }
                // output
                if constexpr (F32) {
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int e = 0; e < NV; ++e)
                                o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[s][j][e]), pw[4 * s + j], o[e], 0, 0, 0);
                } else {
                    typename Kv16<T>::Frag pf[Kv16<T>::PIECES];
                    split_pieces<T>(pw, pf);
#pragma unroll
                    for (int e = 0; e < NV; ++e) {
                        int4 a;
                        int* ap = reinterpret_cast<int*>(&a);
#pragma unroll
                        for (int d = 0; d < 4; ++d)         // slots 2d, 2d + 1: rows (half d / 2, 2 (d % 2)) and the next
                            ap[d] = __builtin_amdgcn_perm(vr[d >> 1][2 * (d & 1) + 1][e >> 1], vr[d >> 1][2 * (d & 1)][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
                        const auto vf = __builtin_bit_cast(typename Kv16<T>::Frag, a);
#pragma unroll
                        for (int n = Kv16<T>::PIECES - 1; n >= 0; --n) o[e] = Kv16<T>::mfma(vf, pf[n], o[e]);
                    }
                }
                load_v();
            }
        }

        // ---- the waves' shares meet
        l += lane_xor16(l);
        l += lane_xor32(l);
        if (live) {
            if (g == 0) { m_s[wave][i] = m; l_s[wave][i] = l; }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < NV; e += NV < 4 ? NV : 4) {
                    float* at = &o_s[wave][i][feature_of<DH, sizeof(T)>(4 * g + j, e)];
                    if constexpr (NV >= 4) *reinterpret_cast<float4*>(at) = make_float4(o[e][j], o[e + 1][j], o[e + 2][j], o[e + 3][j]);
                    else *reinterpret_cast<float2*>(at) = make_float2(o[e][j], o[e + 1][j]);
                }
        }
        __syncthreads();
        join_waves<NW, 16, DH>(p, u, seg, ws, o_s, m_s, l_s);
        if (SPLIT && part.left > 0) __syncthreads();         // (before the next segment's shares)
    } while (SPLIT && part.left > 0);
}

// The same for a key head that only one query head reads, or two of float32 (NQ): most columns of a matrix tile would be empty, and its 64
// float32 matrix instructions a tile (2048 cycles) or the pieces of 16-bit ones would set the time of a short request.  On the vector ALU a tile
// is 64 multiply-adds, 32 data-parallel additions and 8 exponentials a lane and query (some 700 cycles).  Lane (i, g) holds the
// depth/16 features of rows 4g + j of a half that feature_of says, of K as of V; the sixteen lanes of a row add up its score.
// One request of 1000 rows, 4 key heads of 64 and of 128, matrix cores / here: one query head each 12.8 / 6.7 and 21.2 / 10.4 us, two 12.9 / 8.9
// and 21.5 / 12.0; 64 such requests, bound by memory: 22.0 / 21.2 and 43.2 / 42.9, two 22.1 / 23.2 and 43.2 / 43.8 us (6.1 TB/s).  bfloat16, 4 key
// heads of 32 / 64 / 128, one query head each: one request of 400 rows 4.8 / 4.2, 5.4 / 5.1 and 7.3 / 6.2 us, 128 of 1000 12.8 / 13.7, 21.9 / 23.4 and
// 43.9 / 43.8; two query heads each: 4.8 / 5.3, 5.4 / 6.6 and 7.4 / 8.4, 12.8 / 16.0, 22.2 / 24.1 and 44.3 / 46.9, so the matrix cores keep those.
__device__ __forceinline__ float row_sum(float v) {     // over the 16 lanes of a row, to all of them
#define ESTTS_ROW_STEP(ctrl) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, false))
    ESTTS_ROW_STEP(0xB1);        // quad_perm [1, 0, 3, 2]
    ESTTS_ROW_STEP(0x4E);        // quad_perm [2, 3, 0, 1]
    ESTTS_ROW_STEP(0x141);       // row_half_mirror
    ESTTS_ROW_STEP(0x140);       // row_mirror
#undef ESTTS_ROW_STEP
    return v;
}

template <typename T, int DH, bool MASK, bool STREAM, bool SPLIT, int NQ, int NW>
__global__ __launch_bounds__(NW * 64, 2) void paged_attention_few_kernel(const estts_paged_attention_args p, const PagedCall c) {
    constexpr int ES = (int)sizeof(T), HALVES = tile_halves(DH, ES), TILE = 16 * HALVES;
    constexpr uint32_t ALL_ROWS = HALVES == 2 ? 0xFFFFFFFFu : 0xFFFFu;
    constexpr int NV = DH / 16, RUN = NV * ES < 16 ? NV : 16 / ES, RUNS = NV / RUN;        // features of a row per lane, of one load
    typedef __attribute__((ext_vector_type(RUN))) T run_t;
    __shared__ __attribute__((aligned(16))) float o_s[NW][NQ][DH];
    __shared__ float m_s[NW][NQ], l_s[NW][NQ];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedUnit<NQ> u(p, c);
    const PagedScratch ws(p.ws, c.target, p.H, DH);
    PagedPart<NW * 64, TILE * NW, SPLIT> part;
    if (!part.find(p, c, u.part)) return;
    do {
        const PagedSegment seg = part.next(p, u.h0 == 0 && threadIdx.x == 0 ? ws.items : nullptr);
        const int b = seg.b, begin = seg.begin, end = seg.end;
        PageWalk<HALVES, NW> walk(p, c, b, begin, wave, ES);
        const float qs = p.scale * 1.4426950408889634f;
        float qx[NQ][NV];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int e = 0; e < NV; ++e) qx[n][e] = p.q[b * p.ldq + (long)(u.h0 + min(n, u.heads - 1)) * DH + feature_of<DH, ES>(i, e)] * qs;
        const int n_tiles = (end - begin + TILE - 1) / TILE;
        const int n_mine = __builtin_amdgcn_readfirstlane(n_tiles > wave ? (n_tiles - wave + NW - 1) / NW : 0);
        const char* kbase = static_cast<const char*>(p.k_cache) + u.hk * p.s_head * ES;
        const char* vbase = static_cast<const char*>(p.v_cache) + u.hk * p.s_head * ES;
        const int row_bytes = (int)(p.s_row * ES);
        int lane_at = 4 * g * row_bytes + i * ES * RUN;      // (0 behind the last tile: one line for the whole wave)

        run_t kr[HALVES][4][RUNS], vr[HALVES][4][RUNS];
        [[maybe_unused]] float mk;
        auto load = [&](const char* base, run_t (&r)[HALVES][4][RUNS], auto hint) {
#pragma unroll
            for (int s = 0; s < HALVES; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int x = 0; x < RUNS; ++x) {
                        const run_t* at = reinterpret_cast<const run_t*>(base + walk.at[s] + (unsigned)(lane_at + 16 * ES * RUN * x + j * row_bytes));
                        if constexpr (decltype(hint)::value) r[s][j][x] = __builtin_nontemporal_load(at);
                        else r[s][j][x] = *at;
                    }
        };
        auto load_k = [&]() { load(kbase, kr, std::false_type()); };
        auto load_v = [&]() { load(vbase, vr, std::bool_constant<STREAM>()); };
        auto load_mask = [&](int it) {
            if constexpr (MASK) mk = p.key_mask[b * p.mask_sb + min(begin + (it * NW + wave) * TILE + lane % TILE, end - 1) * p.mask_ss];
        };
        float m[NQ], l[NQ], o[NQ][NV];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.0f;
#pragma unroll
            for (int e = 0; e < NV; ++e) o[n][e] = 0.0f;
        }
        if (n_mine > 0) {
            walk.locate(0, false);
            load_k();
            load_mask(0);
            load_v();
            for (int it = 0; it < n_mine; ++it) {
                const int r0 = begin + (it * NW + wave) * TILE;
                bool ok_now[HALVES], all_in = r0 + TILE <= end;
#pragma unroll
                for (int s = 0; s < HALVES; ++s) {
                    ok_now[s] = walk.ok[s];
                    all_in = all_in && ok_now[s];
                }
                float sc[NQ][HALVES][4];
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float t = (float)kr[s][j][0][0] * qx[n][0];
#pragma unroll
                            for (int e = 1; e < NV; ++e) t = fmaf((float)kr[s][j][e / RUN][e % RUN], qx[n][e], t);
                            sc[n][s][j] = row_sum(t);
                        }
                uint32_t rows_in = 0;
                bool drop = !all_in;
                if (MASK || drop) {
                    rows_in = rows_that_count<HALVES>(r0, end, ok_now, MASK ? mk : 0.0f);
                    drop = rows_in != ALL_ROWS;
                }
                const int nx = min(it + 1, n_mine - 1);
                walk.locate(nx, nx != it);
                if (nx == it) lane_at = 0;
                load_k();
                load_mask(nx);
                if (drop) {
                    const uint32_t mine = rows_in >> (4 * g);
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const bool in = mine >> (16 * s + j) & 1;
#pragma unroll
                            for (int n = 0; n < NQ; ++n) sc[n][s][j] = in ? sc[n][s][j] : -INFINITY;
#pragma unroll
                            for (int x = 0; x < RUNS; ++x)
                                if (!in) vr[s][j][x] = (run_t)(T)0.0f;
                        }
                }
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    float top = sc[n][0][0];
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) top = fmaxf(top, sc[n][s][j]);
                    top = fmaxf(top, lane_xor16(top));
                    top = fmaxf(top, lane_xor32(top));
                    const float m1 = fmaxf(m[n], top);
                    const float base = m1 == -INFINITY ? 0.0f : m1;
                    const float c = __builtin_amdgcn_exp2f(m[n] - base);
                    m[n] = m1;
                    l[n] *= c;
#pragma unroll
                    for (int e = 0; e < NV; ++e) o[n][e] *= c;
#pragma unroll
                    for (int s = 0; s < HALVES; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float w = __builtin_amdgcn_exp2f(sc[n][s][j] - base);
                            l[n] += w;
#pragma unroll
                            for (int e = 0; e < NV; ++e) o[n][e] = fmaf(w, (float)vr[s][j][e / RUN][e % RUN], o[n][e]);
                        }
                }
                load_v();
            }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            l[n] += lane_xor16(l[n]);
            l[n] += lane_xor32(l[n]);
            if (lane == 0) { m_s[wave][n] = m[n]; l_s[wave][n] = l[n]; }
#pragma unroll
            for (int e = 0; e < NV; ++e) {
                o[n][e] += lane_xor16(o[n][e]);
                o[n][e] += lane_xor32(o[n][e]);
                if (g == 0) o_s[wave][n][feature_of<DH, ES>(i, e)] = o[n][e];
            }
        }
        __syncthreads();
        join_waves<NW, NQ, DH>(p, u, seg, ws, o_s, m_s, l_s);
        if (SPLIT && part.left > 0) __syncthreads();         // (before the next segment's shares)
    } while (SPLIT && part.left > 0);
}

// The parts of a request meet: one workgroup per (query head, request).  Each of its eight half-waves takes every eighth part, four at a
// time and each read once, with a running maximum of its own; then they meet in the LDS.
template <int DH>
__global__ __launch_bounds__(256) void paged_join_kernel(const estts_paged_attention_args p, const int target) {
    __shared__ float acc_s[8][DH], m_s[8], l_s[8];
    const int h = blockIdx.x, b = blockIdx.y;
    const int lane = threadIdx.x & 31, team = threadIdx.x >> 5;
    const PagedScratch ws(p.ws, target, p.H, DH);
    const int2 it = ws.items[b];
    if (it.y <= 1) return;
    constexpr int PER = DH / 32, STEP = 4;            // features per lane; parts in flight
    float acc[PER] = {}, m = -INFINITY, l = 0.0f;
    for (int s0 = team; s0 < it.y; s0 += 8 * STEP) {
        float2 ml[STEP];
        float x[STEP][PER];
#pragma unroll
        for (int k = 0; k < STEP; ++k) {
            // part it.x holds the request's beginning (place 2 it.x + 1), the others are at the even places after it
            const int s = min(s0 + 8 * k, it.y - 1);
            const long at = (long)(s == 0 ? 2 * it.x + 1 : 2 * (it.x + s)) * p.H + h;
            ml[k] = ws.ml[at];
#pragma unroll
            for (int e = 0; e < PER; ++e) x[k][e] = ws.out[at * DH + lane * PER + e];
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < STEP; ++k) {
            if (s0 + 8 * k >= it.y) ml[k] = make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, ml[k].x);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        const float c0 = __builtin_amdgcn_exp2f(m - base);
        l *= c0;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] *= c0;
#pragma unroll
        for (int k = 0; k < STEP; ++k) {
            const float c = __builtin_amdgcn_exp2f(ml[k].x - base);
            l = fmaf(ml[k].y, c, l);
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] = fmaf(x[k][e], c, acc[e]);
        }
        m = top;
    }
    if (lane == 0) { m_s[team] = m; l_s[team] = l; }
#pragma unroll
    for (int e = 0; e < PER; ++e) acc_s[team][lane * PER + e] = acc[e];
    __syncthreads();
    for (int d = threadIdx.x; d < DH; d += 256) {
        float top = -INFINITY, sum = 0.0f, a = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, m_s[k]);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float c = __builtin_amdgcn_exp2f(m_s[k] - base);
            sum = fmaf(l_s[k], c, sum);
            a = fmaf(acc_s[k][d], c, a);
        }
        p.ctx[b * p.ldo + (long)h * DH + d] = sum == 0.0f ? 0.0f : a / sum;
    }
}

// How many parts a call is cut into (0: one workgroup per request and key head, one launch).
// Parts: one workgroup per CU.  Its four waves keep 64 KB of keys and values in flight, and more parts are more ends to join (256 / 512 / 1024
// parts over all key heads: 61 ragged requests up to 4096 rows of bfloat16 89.3 / 90.0 / 92.4 us, one of 131071 rows 86.2 / 87.5 / 90.5; 128
// leave half of the CUs idle: 121.1 and 106.1).
// Requests of up to 1024 rows are not cut: the second launch costs what the shorter sweep gains (4 heads of 64, float32, cut / not cut: one
// request of 600 rows 6.2 / 5.1 us, of 1000 6.4 / 6.7; and a launch less to issue).  But few wide ones are, from 512 KB a key head on, or
// 256 KB where the matrix cores have more to do to a row (4 heads of 128, float32: one request of 500 rows 6.6 / 6.7 us, of 1000 6.5 / 10.4, eight
// ragged ones 9.8 / 12.9, sixteen 12.9 / 13.5 and of 600 11.0 / 9.7; 32 heads on 8 of 128, bfloat16: one of 450 rows 8.0 / 7.9, of 1000 8.2 / 12.3,
// eight 12.4 / 13.0, sixteen 16.1 / 13.5).  Nor are requests of up to 2048 cut where there is a workgroup for every CU and no second round of
// many (32 heads on 8 of 128, bfloat16, cut / not cut: 32 requests of 2000 45.3 / 43.4 us, 32 ragged ones 28.3 / 28.0; but 128 166.7 / 161.3
// and 128 ragged ones 93.7 / 103.0, 256 177.3 / 179.8).
int paged_split_target(int B, int H, int kv_heads, int depth, int max_len, int type) {
    const long per = (long)kv_heads * ((H / kv_heads + 15) / 16), units = B * per;
    const int esize = type == ESTTS_KV_F32 ? 4 : 2;
    const bool matrix = H > few_queries(esize) * kv_heads;
    const bool heavy = units <= (matrix ? 64 : 32) && 2LL * max_len * depth * esize > (matrix ? 256 : 512) * 1024;
    if ((max_len <= 1024 && !heavy) || (units >= 256 && units < 1024 && max_len <= 2048)) return 0;
    return per < 256 ? (int)(256 / per) : 1;
}

// Whether the rows are too many for the 256 MB behind the L2s to hold them until the next call, by the most that the lengths can be.
// Plain / streaming loads of V: 32 heads on 8 of 128, bfloat16, 32 requests of 1000 rows (131 MB) 26.3 / 22.4 us, of 2000 48.1 / 43.4, 61
// ragged ones up to 4096 (512 MB) 98.4 / 89.3, one of 131071 (537 MB) 96.0 / 86.2 (6.2 TB/s); 8 heads of 64, float32, 200 of 1021 (836 MB)
// 145.9 / 130.9 (6.4 TB/s).  But 32 ragged ones up to 1000 (65 MB, called again and again) 15.4 / 16.4, 8 float32 ones of 1000, 4 heads of 64
// (16 MB), 8.5 / 10.7.
bool stream_rows(const estts_paged_attention_args& a) {
    return 2.0 * a.B * a.max_len * a.kv_heads * a.depth * (a.type == ESTTS_KV_F32 ? 4 : 2) > 100e6;
}

bool bad_cache(const void* k, const void* v, int64_t s_page, int64_t s_head, int64_t s_row, int type, int depth) {
    const int per16 = type == ESTTS_KV_F32 ? 4 : 8;
    return !k || !v || (reinterpret_cast<uintptr_t>(k) & 15) || (reinterpret_cast<uintptr_t>(v) & 15) || s_page % per16 || s_head % per16 ||
           s_row % per16 || s_row < depth || s_page < 0 || s_head < 0;
}

}  // namespace

constexpr int PLAN_ROWS = 4096;        // rows from which the copies of a plan are a launch of their own

extern "C" int64_t estts_page_plan_ws_bytes(int32_t B, int32_t T) {
    return B > PLAN_LDS || T > PLAN_ROWS ? 4 * (PLAN_HEAD + 4 * (int64_t)B) : 0;
}

template <bool PADDED, bool SPLIT>
static void launch_page_scans(const estts_page_plan_args& a, const PageDivisors& by, hipStream_t st) {
    if (a.B > PLAN_LDS) ESTTS_LAUNCH((page_plan_kernel<1024, false, PADDED, SPLIT>), dim3(1), dim3(1024), 0, st, a, by);
    else if (a.B > 256 || (!SPLIT && a.T > 1024)) ESTTS_LAUNCH((page_plan_kernel<1024, true, PADDED, SPLIT>), dim3(1), dim3(1024), 0, st, a, by);
    else ESTTS_LAUNCH((page_plan_kernel<256, true, PADDED, SPLIT>), dim3(1), dim3(256), 0, st, a, by);
}

template <bool PADDED>
static void launch_page_plan(const estts_page_plan_args& a, hipStream_t st) {
    const PageDivisors by = {page_size(a.page), divisor(PADDED ? a.R : 1, 30)};
    if (a.T <= PLAN_ROWS) return launch_page_scans<PADDED, false>(a, by, st);
    launch_page_scans<PADDED, true>(a, by, st);
    // (threads enough for the rows, for the pages that they may take and for those that may come back)
    const long wgs = ((long)a.T + a.T / a.page + a.B + a.n_pages + 255) / 256;
    const dim3 grid((unsigned)(wgs < 1024 ? wgs : 1024));
    if (a.B > PLAN_LDS) ESTTS_LAUNCH((page_copy_kernel<false, PADDED>), grid, dim3(256), 0, st, a, by);
    else ESTTS_LAUNCH((page_copy_kernel<true, PADDED>), grid, dim3(256), 0, st, a, by);
}

extern "C" int estts_page_plan(const estts_page_plan_args* args, void* stream) {
    ESTTS_CHECK_ARG(args != nullptr, "estts_page_plan: null args");
    const estts_page_plan_args& a = *args;
    ESTTS_CHECK_ARG(a.lengths && a.n_new && a.block_table && a.free_pages && a.n_free && a.slots && a.lengths_out && a.n_free_out,
                    "estts_page_plan: null pointer");
    ESTTS_CHECK_ARG(a.B > 0 && a.P > 0 && a.n_pages > 0 && a.T > 0 && a.T < (1 << 30) && a.R >= 0 && a.ld_table >= a.P,
                    "estts_page_plan: bad shape");
    ESTTS_CHECK_ARG(a.R == 0 || (int64_t)a.B * a.R == a.T, "estts_page_plan: a padded slot map holds B * R entries");
    ESTTS_CHECK_ARG(a.page > 0 && a.page % 16 == 0, "estts_page_plan: page must be a multiple of 16 (got %d)", a.page);
    ESTTS_CHECK_ARG((int64_t)a.P * a.page < (1LL << 31) && (int64_t)a.n_pages * a.page < (1LL << 31) && (int64_t)a.B * a.P < (1LL << 31),
                    "estts_page_plan: P * page, n_pages * page and B * P must stay below 2^31");
    const int64_t need = estts_page_plan_ws_bytes(a.B, a.T);
    ESTTS_CHECK_ARG(need == 0 || (a.ws && a.ws_bytes >= need && !(reinterpret_cast<uintptr_t>(a.ws) & 15)),
                    "estts_page_plan: this call needs %ld bytes of scratch, 16-byte aligned (given: %ld)", (long)need, (long)a.ws_bytes);
    if (a.R) launch_page_plan<true>(a, (hipStream_t)stream);
    else launch_page_plan<false>(a, (hipStream_t)stream);
    ESTTS_CHECK_LAUNCH("estts_page_plan");
    return 0;
}

template <typename T>
static void launch_page_write(const estts_page_write_args& a, hipStream_t stream) {
    const int pieces = a.heads * a.depth / (16 / (int)sizeof(T));
    int log = 0;
    while ((1 << log) < pieces && log < 8) ++log;
    const int rows = 256 >> log, cols = (pieces + (1 << log) - 1) >> log;
    const dim3 grid((unsigned)((a.T + rows - 1) / rows * cols));
    if ((double)a.T * a.heads * a.depth * sizeof(T) * 2 > 16e6)
        ESTTS_LAUNCH((page_write_kernel<T, true>), grid, dim3(256), 0, stream, a, log, cols);
    else
        ESTTS_LAUNCH((page_write_kernel<T, false>), grid, dim3(256), 0, stream, a, log, cols);
}

extern "C" int estts_page_write(const estts_page_write_args* args, void* stream) {
    ESTTS_CHECK_ARG(args != nullptr, "estts_page_write: null args");
    const estts_page_write_args& a = *args;
    ESTTS_CHECK_ARG(a.k && a.v && a.slots, "estts_page_write: null pointer");
    ESTTS_CHECK_ARG(a.T > 0 && a.heads > 0 && a.depth > 0 && a.n_pages > 0, "estts_page_write: bad shape");
    ESTTS_CHECK_ARG(a.depth % 8 == 0 && a.depth <= 1024, "estts_page_write: depth must be a multiple of 8, at most 1024");
    ESTTS_CHECK_ARG((int64_t)a.heads * a.depth <= (1 << 20) && (int64_t)a.T * a.heads * a.depth < (1LL << 32),
                    "estts_page_write: heads * depth must be at most 2^20 and T * heads * depth below 2^32");
    ESTTS_CHECK_ARG(a.page > 0 && a.page % 16 == 0, "estts_page_write: page must be a multiple of 16 (got %d)", a.page);
    ESTTS_CHECK_ARG((int64_t)a.n_pages * a.page < (1LL << 31), "estts_page_write: n_pages * page must stay below 2^31");
    ESTTS_CHECK_ARG(a.type >= ESTTS_KV_F32 && a.type <= ESTTS_KV_F16, "estts_page_write: unknown cache type %d", a.type);
    const int64_t width = (int64_t)a.heads * a.depth;
    ESTTS_CHECK_ARG(!(reinterpret_cast<uintptr_t>(a.k) & 15) && !(reinterpret_cast<uintptr_t>(a.v) & 15) && a.ldk % 4 == 0 && a.ldv % 4 == 0 &&
                    a.ldk >= width && a.ldv >= width, "estts_page_write: rows must be 16-byte aligned and at least heads * depth long");
    ESTTS_CHECK_ARG(!bad_cache(a.k_cache, a.v_cache, a.s_page, a.s_head, a.s_row, a.type, a.depth),
                    "estts_page_write: caches and their strides must be multiples of 16 bytes");
    if (a.type == ESTTS_KV_F32) launch_page_write<float>(a, (hipStream_t)stream);
    else if (a.type == ESTTS_KV_BF16) launch_page_write<__bf16>(a, (hipStream_t)stream);
    else launch_page_write<_Float16>(a, (hipStream_t)stream);
    ESTTS_CHECK_LAUNCH("estts_page_write");
    return 0;
}

extern "C" int64_t estts_paged_attention_ws_bytes(int32_t B, int32_t H, int32_t kv_heads, int32_t depth, int32_t max_len, int32_t type) {
    if (B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads || depth <= 0 || max_len <= 0) return 0;      // (estts_paged_attention says why not)
    const int target = paged_split_target(B, H, kv_heads, depth, max_len, type);
    return target ? PagedScratch::bytes(target, H, depth, B) : 0;
}

template <typename T, int DH, bool MASK, bool STREAM, bool SPLIT>
static void launch_paged_attention(const estts_paged_attention_args& a, int target, hipStream_t stream) {
    const int group = a.H / a.kv_heads, n_group = (group + 15) / 16;
    const int units = (target ? target : a.B) * a.kv_heads;
    const PagedCall c = {page_size(a.page), group, n_group, target, divisor(a.kv_heads, 30), divisor(target ? target : 1, 30)};
    const dim3 grid(n_group > 1 ? (units + 7) / 8 * 8 * n_group : units), block(ATT_WAVES * 64);
    constexpr int NW = SPLIT ? ATT_WAVES : FEW_WAVES;
    constexpr int FEW = few_queries((int)sizeof(T));
    if (group == 1) ESTTS_LAUNCH((paged_attention_few_kernel<T, DH, MASK, STREAM, SPLIT, 1, NW>), grid, dim3(NW * 64), 0, stream, a, c);
    else if (group <= FEW) ESTTS_LAUNCH((paged_attention_few_kernel<T, DH, MASK, STREAM, SPLIT, FEW, NW>), grid, dim3(NW * 64), 0, stream, a, c);
    else ESTTS_LAUNCH((paged_attention_kernel<T, DH, MASK, STREAM, SPLIT, ATT_WAVES>), grid, block, 0, stream, a, c);
}

template <typename T, int DH, bool SPLIT>
static void launch_paged_attention(const estts_paged_attention_args& a, int target, hipStream_t stream) {
    const bool many = stream_rows(a);
    if (a.key_mask && many) launch_paged_attention<T, DH, true, true, SPLIT>(a, target, stream);
    else if (a.key_mask) launch_paged_attention<T, DH, true, false, SPLIT>(a, target, stream);
    else if (many) launch_paged_attention<T, DH, false, true, SPLIT>(a, target, stream);
    else launch_paged_attention<T, DH, false, false, SPLIT>(a, target, stream);
    if (SPLIT) ESTTS_LAUNCH(paged_join_kernel<DH>, dim3(a.H, a.B), dim3(256), 0, stream, a, target);
}

template <typename T, int DH>
static void launch_paged_attention(const estts_paged_attention_args& a, int target, hipStream_t stream) {
    if (target) launch_paged_attention<T, DH, true>(a, target, stream);
    else launch_paged_attention<T, DH, false>(a, target, stream);
}

template <typename T>
static void launch_paged_attention(const estts_paged_attention_args& a, int target, hipStream_t stream) {
    if (a.depth == 32) launch_paged_attention<T, 32>(a, target, stream);
    else if (a.depth == 64) launch_paged_attention<T, 64>(a, target, stream);
    else launch_paged_attention<T, 128>(a, target, stream);
}

extern "C" int estts_paged_attention(const estts_paged_attention_args* args, void* stream) {
    ESTTS_CHECK_ARG(args != nullptr, "estts_paged_attention: null args");
    estts_paged_attention_args a = *args;
    ESTTS_CHECK_ARG(a.q && a.block_table && a.lengths && a.ctx, "estts_paged_attention: null pointer");
    ESTTS_CHECK_ARG(a.B > 0 && a.B <= 65535 && a.H > 0 && a.kv_heads > 0 && a.H % a.kv_heads == 0 && a.P > 0 && a.n_pages > 0 && a.ld_table >= a.P,
                    "estts_paged_attention: bad shape (B 1 .. 65535, heads a multiple of kv_heads)");
    ESTTS_CHECK_ARG(a.depth == 32 || a.depth == 64 || a.depth == 128, "estts_paged_attention: depth must be 32, 64 or 128 (got %d)", a.depth);
    ESTTS_CHECK_ARG(a.page > 0 && a.page % 16 == 0, "estts_paged_attention: page must be a multiple of 16 (got %d)", a.page);
    ESTTS_CHECK_ARG((int64_t)a.P * a.page <= (1LL << 30) && (int64_t)a.n_pages * a.page < (1LL << 31),
                    "estts_paged_attention: P * page must be at most 2^30, n_pages * page below 2^31");
    ESTTS_CHECK_ARG(a.type >= ESTTS_KV_F32 && a.type <= ESTTS_KV_F16, "estts_paged_attention: unknown cache type %d", a.type);
    const int64_t width = (int64_t)a.H * a.depth;
    ESTTS_CHECK_ARG(!(reinterpret_cast<uintptr_t>(a.q) & 15) && a.ldq % 4 == 0 && a.ldq >= width && a.ldo >= width,
                    "estts_paged_attention: query rows must be 16-byte aligned, rows at least H * depth long");
    ESTTS_CHECK_ARG(!bad_cache(a.k_cache, a.v_cache, a.s_page, a.s_head, a.s_row, a.type, a.depth),
                    "estts_paged_attention: caches and their strides must be multiples of 16 bytes");
    ESTTS_CHECK_ARG(a.s_row * (int64_t)a.page < (1LL << 28), "estts_paged_attention: the rows of one page must span less than 2^28 elements");
    ESTTS_CHECK_ARG(a.max_len >= 0, "estts_paged_attention: max_len must not be negative");
    if (a.max_len == 0 || (int64_t)a.max_len > (int64_t)a.P * a.page) a.max_len = a.P * a.page;
    ESTTS_CHECK_ARG((int64_t)a.B * a.max_len < (1LL << 36) && (int64_t)a.B * a.H < (1LL << 23),
                    "estts_paged_attention: B * max_len must stay below 2^36 and B * H below 2^23");
    const int target = paged_split_target(a.B, a.H, a.kv_heads, a.depth, a.max_len, a.type);
    const int64_t need = target ? PagedScratch::bytes(target, a.H, a.depth, a.B) : 0;
    ESTTS_CHECK_ARG(need == 0 || (a.ws && a.ws_bytes >= need && !(reinterpret_cast<uintptr_t>(a.ws) & 15)),
                    "estts_paged_attention: this call needs %ld bytes of scratch, 16-byte aligned (given: %ld)", (long)need, (long)a.ws_bytes);
    if (a.type == ESTTS_KV_F32) launch_paged_attention<float>(a, target, (hipStream_t)stream);
    else if (a.type == ESTTS_KV_BF16) launch_paged_attention<__bf16>(a, target, (hipStream_t)stream);
    else launch_paged_attention<_Float16>(a, target, (hipStream_t)stream);
    ESTTS_CHECK_LAUNCH("estts_paged_attention");
    return 0;
}
