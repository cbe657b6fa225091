// Paged key / value memory: the page plan of a step, the write of new rows into the pages, the attention of one new row per
// request over its pages (see estts_page_plan, estts_page_write, estts_paged_attention in include/estts.h).
#include "common.h"

#include <type_traits>

namespace {

// ------------------------------------------------------------------------------------------------ page plan
constexpr int PLAN_THREADS = 1024;

__device__ __forceinline__ int pages_of(int rows, int page) { return (int)(((unsigned)rows + page - 1) / (unsigned)page); }

// inclusive prefix sum over the workgroup's threads, and the total
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* part, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const V up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    __syncthreads();                       // (the last scan's readers of part are done)
    if (lane == 63) part[wave] = v;
    __syncthreads();
    V before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 64; ++w) {
        const V s = part[w];
        if (w < wave) before += s;
        total += s;
    }
    return v + before;
}

// first b with end[b] > x (ends do not decrease); B if there is none
__device__ __forceinline__ int first_past(const int* end, int B, int x) {
    int lo = 0, hi = B;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// One workgroup.  ws holds per request: end of its rows in a packed slot map (at most T), pages granted up to and including it, and its
// length (complemented where it gets no rows).
__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(const estts_page_plan_args p) {
    __shared__ int part_i[16];
    __shared__ long long part_l[16];
    const int tid = threadIdx.x;
    const int cap = p.P * p.page;
    int* const row_end = p.ws;
    int* const page_end = p.ws + p.B;
    int* const len_of = p.ws + 2 * (long)p.B;

    const int height0 = min(max(p.n_free[0], 0), p.n_pages);
    // 1. pages of the requests that ended
    int back = 0;
    for (int b0 = 0; b0 < p.B; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        const bool ended = b < p.B && p.n_new[b] < 0;
        const int used = ended ? pages_of(min(max(p.lengths[b], 0), cap), p.page) : 0;
        int total;
        const int upto = block_scan(used, part_i, total);
        if (b < p.B) page_end[b] = back + upto;
        back += total;
    }
    __syncthreads();
    back = min(back, p.n_pages - height0);          // (more would be pages that are held twice)
    for (int g = tid; g < back; g += PLAN_THREADS) {
        const int b = first_past(page_end, p.B, g);
        const int j = g - (b ? page_end[b - 1] : 0);
        p.free_pages[height0 + g] = p.block_table[b * p.ld_table + j];
    }
    const int height = height0 + back;
    __syncthreads();
    // 2. grants
    int asked = 0, taken = 0, refused = 0;
    long long rows = 0;
    for (int b0 = 0; b0 < p.B; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        const int n = b < p.B ? p.n_new[b] : 0;
        const int len = b < p.B ? min(max(p.lengths[b], 0), cap) : 0;
        const long long want = max(n, 0);
        long long rows_total;
        const long long rows_upto = rows + block_scan(want, part_l, rows_total);
        const bool fits = b < p.B && n >= 0 && len + want <= cap && (want == 0 || (p.R ? want <= p.R : rows_upto <= p.T));
        const int need = fits ? pages_of(len + (int)want, p.page) - pages_of(len, p.page) : 0;
        int need_total;
        const int upto = asked + block_scan(need, part_i, need_total);
        const bool granted = fits && (need == 0 || upto <= height);
        int refused_total, taken_total;
        block_scan((int)(b < p.B && n >= 0 && !granted), part_i, refused_total);
        block_scan(granted ? need : 0, part_i, taken_total);
        if (b < p.B) {
            row_end[b] = (int)min(rows_upto, (long long)p.T);
            page_end[b] = min(upto, height);        // (a request that is turned away ends no page below its own)
            len_of[b] = granted ? len : ~len;
            p.lengths_out[b] = n < 0 ? 0 : granted ? len + (int)want : len;
        }
        rows += rows_total;
        asked += need_total;
        taken += taken_total;
        refused += refused_total;
    }
    __syncthreads();
    for (int g = tid; g < taken; g += PLAN_THREADS) {
        const int b = first_past(page_end, p.B, g);
        const int i = g - (b ? page_end[b - 1] : 0);
        p.block_table[b * p.ld_table + pages_of(len_of[b], p.page) + i] = p.free_pages[height - 1 - g];
    }
    if (tid == 0) {
        p.n_free_out[0] = height - taken;
        if (p.refused) p.refused[0] = refused;
    }
    __syncthreads();
    // 3. where each row goes
    for (int t = tid; t < p.T; t += PLAN_THREADS) {
        const int b = p.R ? t / p.R : first_past(row_end, p.B, t);
        int slot = -1, pos = -1;
        if (b < p.B && len_of[b] >= 0) {
            const int i = p.R ? t - b * p.R : t - (b ? row_end[b - 1] : 0);
            if (!p.R || i < p.n_new[b]) {
                pos = len_of[b] + i;
                const int id = p.block_table[b * p.ld_table + pos / p.page];
                if (id >= 0 && id < p.n_pages) slot = id * p.page + pos % p.page;
            }
        }
        p.slots[t] = slot;
        if (p.positions) p.positions[t] = pos;
    }
}

// ------------------------------------------------------------------------------------------------ rows into the pages
template <typename T>
struct Vec4 { T v[4]; };

template <typename T>
__global__ __launch_bounds__(256) void page_write_kernel(const estts_page_write_args p) {
    const int per = p.heads * (p.depth >> 2);                  // four-element pieces of a row
    const long total = (long)p.T * per;
    const long limit = (long)p.n_pages * p.page;
    for (long x = (long)blockIdx.x * 256 + threadIdx.x; x < total; x += (long)gridDim.x * 256) {
        const int t = (int)(x / per), c = (int)(x - (long)t * per) << 2;
        const int slot = p.slots[t];
        if (slot < 0 || slot >= limit) continue;
        const int h = c / p.depth, d = c - h * p.depth;
        const long at = (long)(slot / p.page) * p.s_page + (long)h * p.s_head + (long)(slot % p.page) * p.s_row + d;
        const float4 kx = *reinterpret_cast<const float4*>(p.k + t * p.ldk + c), vx = *reinterpret_cast<const float4*>(p.v + t * p.ldv + c);
        *reinterpret_cast<Vec4<T>*>(static_cast<T*>(p.k_cache) + at) = {(T)kx.x, (T)kx.y, (T)kx.z, (T)kx.w};
        *reinterpret_cast<Vec4<T>*>(static_cast<T*>(p.v_cache) + at) = {(T)vx.x, (T)vx.y, (T)vx.z, (T)vx.w};
    }
}

// ------------------------------------------------------------------------------------------------ attention of one new row
// With t = scale log2(e) q . k_j and M = max_j t_j:  ctx = sum_j 2^(t_j - M) v_j / sum_j 2^(t_j - M), computed in one pass over the rows with a
// running maximum.  What has to move is the keys and values themselves, a few operations per byte: the kernel is laid out so that the
// loads never wait for the arithmetic and the arithmetic stays off the LDS.
//
// A wave sweeps tiles of 16 (float32, depth 128) or 32 rows for up to 16 query heads that share a key head, on the matrix cores:
//   S^T (16 rows x 16 queries) = K Q^T      A = K: lane (i, g) holds row i, elements 8g .. 8g+7 of a step of 32 (float32: 4g .. 4g+3 of 16)
//   O^T (16 features x 16 queries) += V^T P^T   A = V^T: row r of the result is feature r * depth/16 + e in tile e, so that lane i loads the
//       depth/16 consecutive features of a row that it feeds to all tiles, and a row of V is one coalesced load of 16 lanes
// The result layout D[4g + j][i] puts the weights of rows 4g + j into lane (i, g), which is where the second product wants them: of
// two 16-row halves (16-bit types: k slot 8g + 4 half + j is row 16 half + 4g + j) or as they are (float32: k slot g).  Nothing crosses
// lanes but the maximum.  16-bit values of V are interleaved from rows to features with one v_perm_b32 per two values.
// The matrix cores round nothing here that float32 would keep: float32 pages run through the float32 instructions; for 16-bit pages
// the queries and the weights are split into bfloat16 pieces (three, 24 bits) or float16 pieces (two, 22 bits, behind a power of two that
// puts the largest element of the query at 2^13 and the largest weight at 2^14), whose products with the pages' values are exact.
// Scores, maxima, sums and outputs are float32.

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;

constexpr int ATT_WAVES = 4;

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

// x = sum of the pieces up to 2^-24 (bfloat16) or 2^-22 (float16) of x
template <typename T>
__device__ __forceinline__ void split_pieces(const float (&x)[8], typename Kv16<T>::Frag (&f)[Kv16<T>::PIECES]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int n = 0; n < Kv16<T>::PIECES; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const T h = (T)r[e];
            f[n][e] = h;
            r[e] -= (float)h;
        }
}

// The share of the work that workgroup `item` of a key head does: rows [begin, end) of request b, split `split` of `n_split`
struct PagedWork { int b, begin, end, split, n_split, first; bool any; };

__device__ __forceinline__ int request_rows(const estts_paged_attention_args& p, int b) {
    return min(min(max(p.lengths[b], 0), p.P * p.page), p.max_len);
}

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Rows are dealt out in chunks of equal size over all requests, so that long and short requests keep the chip equally busy: about
// `target` chunks, each request at least one, so at most target + B items (the grid).  Every wave finds its own from the lengths.
__device__ __forceinline__ PagedWork find_work(const estts_paged_attention_args& p, int item, int target, int min_rows) {
    PagedWork w;
    if (target == 0) {
        w.b = item; w.begin = 0; w.end = request_rows(p, item); w.split = 0; w.n_split = 1; w.first = item; w.any = true;
        return w;
    }
    const int lane = threadIdx.x & 63;
    constexpr int UNIT = 32 * ATT_WAVES;            // one round of the workgroup's waves over tiles of 32 rows
    int units = 0;                                  // (at most 2^31 / 128 a request: the caller keeps B * P * page / 128 below 2^31)
    for (int b = lane; b < p.B; b += 64) units += (request_rows(p, b) + UNIT - 1) / UNIT;
    units = wave_sum_int(units);
    const int chunk = max((units + target - 1) / target, min_rows / UNIT) * UNIT;
    w.any = false;
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int rows = b0 + lane < p.B ? request_rows(p, b0 + lane) : 0;
        const int n = b0 + lane < p.B ? max((rows - 1) / chunk + 1, 1) : 0;
        int upto = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(upto, d);
            if (lane >= d) upto += up;
        }
        const uint64_t past = __ballot(before + upto > item);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            w.b = b0 + l;
            w.n_split = __shfl(n, l);
            w.first = before + __shfl(upto, l) - w.n_split;
            w.split = item - w.first;
            const int len = __shfl(rows, l);
            w.begin = w.split * chunk;
            w.end = min(len, w.begin + chunk);
            w.any = true;
            break;
        }
        before += __shfl(upto, 63);
    }
    return w;
}

// scratch of a split call: per item and query head the unnormalised output (relative to its maximum), then (maximum, sum); per request
// (first item, number of items)
struct PagedScratch {
    float* out; float2* ml; int2* items;
    __host__ __device__ PagedScratch(void* ws, long n_items, int H, int depth) {
        out = static_cast<float*>(ws);
        ml = reinterpret_cast<float2*>(out + n_items * H * depth);
        items = reinterpret_cast<int2*>(ml + n_items * H);
    }
    static __host__ __device__ long bytes(long n_items, int H, int depth, int B) { return n_items * H * (depth + 2) * 4 + (long)B * 8; }
};

template <typename T, int DH, bool MASK>
__global__ __launch_bounds__(ATT_WAVES * 64, 2) void paged_attention_kernel(const estts_paged_attention_args p, const int target, const int min_rows) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int HALVES = F32 && DH == 128 ? 1 : 2;    // 16-row halves of a tile (float32 at depth 128: 64 registers of K and V are enough in flight)
    constexpr int TILE = 16 * HALVES;
    constexpr int NV = DH / 16;                         // consecutive features of a row of V per lane = tiles of 16 features
    constexpr int PER_BLOCK = 64 / HALVES;              // tiles whose page entries the lanes of the wave hold at once
    __shared__ __attribute__((aligned(16))) float o_s[ATT_WAVES][16][DH];
    __shared__ float m_s[ATT_WAVES][16], l_s[ATT_WAVES][16];

    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // query groups of one key head next to each other on one XCD (workgroups whose numbers agree mod 8), whose L2 then holds the rows
    const int group = p.H / p.kv_heads, n_group = (group + 15) >> 4;
    int unit = blockIdx.x, part = 0;
    if (n_group > 1) {
        const int k = unit >> 3;
        part = k % n_group;
        unit = (k / n_group) * 8 + (unit & 7);
    }
    const int item = unit / p.kv_heads, hk = unit - item * p.kv_heads;
    const int n_items = target ? target + p.B : p.B;
    if (item >= n_items) return;
    const PagedWork w = find_work(p, item, target, min_rows);
    if (!w.any) return;
    const int b = __builtin_amdgcn_readfirstlane(w.b), begin = __builtin_amdgcn_readfirstlane(w.begin), end = __builtin_amdgcn_readfirstlane(w.end);
    const int heads = min(16, group - part * 16);       // query heads of this workgroup
    const int h0 = hk * group + part * 16;

    // ---- queries
    const float qs = p.scale * 1.4426950408889634f;
    const bool live = i < heads;
    const float* qp = p.q + b * p.ldq + (long)(h0 + (live ? i : 0)) * DH;
    constexpr int QV = F32 ? DH / 4 : DH / 4;           // elements of the query per lane
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
    [[maybe_unused]] typename Kv16<typename std::conditional<F32, __bf16, T>::type>::Frag qf[F32 ? 1 : DH / 32][3];
    if constexpr (!F32) {
#pragma unroll
        for (int s = 0; s < DH / 32; ++s) {
            float t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = qx[8 * s + e];
            typename Kv16<T>::Frag f[Kv16<T>::PIECES];
            split_pieces<T>(t, f);
#pragma unroll
            for (int n = 0; n < Kv16<T>::PIECES; ++n) qf[s][n] = f[n];
        }
    }

    // ---- the wave's tiles: t = wave, wave + 4, ... of [begin, end)
    const int n_tiles = (end - begin + TILE - 1) / TILE;
    const int n_mine = __builtin_amdgcn_readfirstlane(n_tiles > wave ? (n_tiles - wave + ATT_WAVES - 1) / ATT_WAVES : 0);
    const int* table = p.block_table + b * p.ld_table;
    const char* kbase = static_cast<const char*>(p.k_cache) + hk * p.s_head * (long)sizeof(T);
    const char* vbase = static_cast<const char*>(p.v_cache) + hk * p.s_head * (long)sizeof(T);
    const int row_bytes = (int)(p.s_row * (long)sizeof(T));
    // first row of half (lane % HALVES) of the wave's tile number block * PER_BLOCK + lane / HALVES; a half lies in one page
    auto half_row = [&](int block) { return begin + ((block * PER_BLOCK + lane / HALVES) * ATT_WAVES + wave) * TILE + (HALVES == 2 ? 16 * (lane & 1) : 0); };
    auto page_entry = [&](int block) { const int r = half_row(block); return r < end ? table[r / p.page] : -1; };
    int entry = page_entry(0), next_entry = page_entry(1);
    int at_lo, at_hi;                                   // byte offset of this lane's half in the caches, -1 where there is no such row or page
    auto place = [&](int block) {
        const int r = half_row(block);
        const bool ok = entry >= 0 && entry < p.n_pages;
        const long at = ok ? ((long)entry * p.s_page + (long)(r % p.page) * p.s_row) * (long)sizeof(T) : -1L;
        at_lo = (int)(at & 0xFFFFFFFFL);
        at_hi = (int)(at >> 32);
    };
    place(0);

    // registers of a tile
    constexpr int KL = F32 ? DH / 16 : DH / 32;         // 16-byte loads of K per half and lane
    constexpr int VW = NV * (int)sizeof(T) / 4;         // dwords of V per row and lane
    int4 kr[HALVES][KL];
    int vr[HALVES][4][VW];
    [[maybe_unused]] float mk[HALVES][4];
    const int k_lane = i * row_bytes + 16 * g;
    const int v_lane = 4 * g * row_bytes + i * NV * (int)sizeof(T);
    long half_at[HALVES];
    bool half_ok[HALVES];
    auto locate = [&](int it) {                         // of tile `it` of the wave
        const int k = it % PER_BLOCK;
#pragma unroll
        for (int s = 0; s < HALVES; ++s) {
            const int lo = __builtin_amdgcn_readlane(at_lo, k * HALVES + s), hi = __builtin_amdgcn_readlane(at_hi, k * HALVES + s);
            half_ok[s] = hi >= 0;
            half_at[s] = hi >= 0 ? (long)(((unsigned long)(unsigned)hi << 32) | (unsigned)lo) : 0;       // (row 0 of page 0 is always there)
        }
    };
    auto load_k = [&](int it) {
#pragma unroll
        for (int s = 0; s < HALVES; ++s) {
            const char* at = kbase + half_at[s];
#pragma unroll
            for (int x = 0; x < KL; ++x) kr[s][x] = *reinterpret_cast<const int4*>(at + (unsigned)(k_lane + 64 * x));
        }
        if constexpr (MASK) {
            const float* mrow = p.key_mask + b * p.mask_sb;
            const int r0 = begin + (it * ATT_WAVES + wave) * TILE + 4 * g;
#pragma unroll
            for (int s = 0; s < HALVES; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) mk[s][j] = mrow[min(r0 + 16 * s + j, end - 1) * p.mask_ss];
        }
    };
    auto load_v = [&](const long (&at_half)[HALVES]) {
#pragma unroll
        for (int s = 0; s < HALVES; ++s) {
            const char* at = vbase + at_half[s];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const char* a = at + (unsigned)(v_lane + j * row_bytes);
                if constexpr (VW >= 4) {
#pragma unroll
                    for (int x = 0; x < VW / 4; ++x) {
                        const int4 t = *reinterpret_cast<const int4*>(a + 16 * x);
                        vr[s][j][4 * x] = t.x; vr[s][j][4 * x + 1] = t.y; vr[s][j][4 * x + 2] = t.z; vr[s][j][4 * x + 3] = t.w;
                    }
                } else if constexpr (VW == 2) {
                    const int2 t = *reinterpret_cast<const int2*>(a);
                    vr[s][j][0] = t.x; vr[s][j][VW - 1] = t.y;
                } else {
                    vr[s][j][0] = *reinterpret_cast<const int*>(a);
                }
            }
        }
    };

    f32x4 o[NV];
#pragma unroll
    for (int e = 0; e < NV; ++e) o[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;                      // of query i; l: this lane's rows only
    constexpr float LIFT = !F32 && sizeof(T) == 2 && std::is_same<T, _Float16>::value ? 14.0f : 0.0f;

    if (n_mine > 0) {
        locate(0);
        load_k(0);
        load_v(half_at);
        bool ok_now[HALVES];
        for (int it = 0; it < n_mine; ++it) {
#pragma unroll
            for (int s = 0; s < HALVES; ++s) ok_now[s] = half_ok[s];
            const int r0 = begin + (it * ATT_WAVES + wave) * TILE;
            // scores
            float sc[HALVES][4];
            if constexpr (F32) {
#pragma unroll
                for (int s = 0; s < HALVES; ++s) {
                    f32x4 a0 = {0.0f, 0.0f, 0.0f, 0.0f}, a1 = a0;
#pragma unroll
                    for (int x = 0; x < KL; ++x) {
                        a0 = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, kr[s][x].x), qx[4 * x], a0, 0, 0, 0);
                        a1 = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, kr[s][x].y), qx[4 * x + 1], a1, 0, 0, 0);
                        a0 = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, kr[s][x].z), qx[4 * x + 2], a0, 0, 0, 0);
                        a1 = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, kr[s][x].w), qx[4 * x + 3], a1, 0, 0, 0);
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
            bool in[HALVES][4];
#pragma unroll
            for (int s = 0; s < HALVES; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    in[s][j] = ok_now[s] && r0 + 16 * s + 4 * g + j < end;
                    if constexpr (MASK) in[s][j] = in[s][j] && mk[s][j] == 0.0f;
                }
            bool drop = !all_in;
            if constexpr (MASK) {
                bool mine = true;
#pragma unroll
                for (int s = 0; s < HALVES; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mine = mine && in[s][j];
                drop = __any(!mine);
            }
            // the next tile's keys, into the registers just read (the last tile again where there is none: the number of loads in
            // flight stays the same on every path, so that no wait is longer than it has to be)
            const int nx = min(it + 1, n_mine - 1);
            if (nx % PER_BLOCK == 0 && nx != it) {
                entry = next_entry;
                place(nx / PER_BLOCK);
                next_entry = page_entry(nx / PER_BLOCK + 1);
            }
            locate(nx);
            load_k(nx);
            if (drop) {
#pragma unroll
                for (int s = 0; s < HALVES; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        sc[s][j] = in[s][j] ? sc[s][j] : -INFINITY;
#pragma unroll
                        for (int x = 0; x < VW; ++x) vr[s][j][x] = in[s][j] ? vr[s][j][x] : 0;       // (0 x NaN would be NaN)
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
            load_v(half_at);
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
                float* at = &o_s[wave][i][(4 * g + j) * NV + e];
                if constexpr (NV >= 4) *reinterpret_cast<float4*>(at) = make_float4(o[e][j], o[e + 1][j], o[e + 2][j], o[e + 3][j]);
                else *reinterpret_cast<float2*>(at) = make_float2(o[e][j], o[e + 1][j]);
            }
    }
    __syncthreads();
    const PagedScratch ws(p.ws, n_items, p.H, DH);
    if (target && w.split == 0 && unit % p.kv_heads == 0 && part == 0 && threadIdx.x == 0) ws.items[b] = make_int2(w.first, w.n_split);
    for (int x = threadIdx.x; x < heads * DH; x += ATT_WAVES * 64) {
        const int h = x / DH, d = x % DH;
        float top = m_s[0][h];
#pragma unroll
        for (int v = 1; v < ATT_WAVES; ++v) top = fmaxf(top, m_s[v][h]);
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int v = 0; v < ATT_WAVES; ++v) {
            const float c = __builtin_amdgcn_exp2f(m_s[v][h] - base);
            sum = fmaf(l_s[v][h], c, sum);
            acc = fmaf(o_s[v][h][d], c, acc);
        }
        if (w.n_split == 1) {
            p.ctx[b * p.ldo + (long)(h0 + h) * DH + d] = sum == 0.0f ? 0.0f : acc / sum;
        } else {
            const long at = (long)item * p.H + h0 + h;
            ws.out[at * DH + d] = acc;
            if (d == 0) ws.ml[at] = make_float2(top, sum);
        }
    }
}

// The splits of a request meet: one workgroup per (query head, request), its waves take every fourth split.
template <int DH>
__global__ __launch_bounds__(256) void paged_join_kernel(const estts_paged_attention_args p, const int n_items) {
    __shared__ float acc_s[4][DH], sum_s[4];
    const int h = blockIdx.x, b = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const PagedScratch ws(p.ws, n_items, p.H, DH);
    const int2 it = ws.items[b];
    if (it.y <= 1) return;
    const float2* ml = ws.ml + (long)it.x * p.H + h;
    float top = -INFINITY;
    for (int s = lane; s < it.y; s += 64) top = fmaxf(top, ml[(long)s * p.H].x);
    top = wave_max(top);
    const float base = top == -INFINITY ? 0.0f : top;
    constexpr int PER = DH / 32;                      // features per lane; the halves of a wave take different splits
    const int f = (lane & 31) * PER;
    float acc[PER] = {}, sum = 0.0f;
    const float* out = ws.out + ((long)it.x * p.H + h) * DH + f;
#pragma unroll 4
    for (int s = 2 * wave + (lane >> 5); s < it.y; s += 8) {
        const float2 v = ml[(long)s * p.H];
        const float c = __builtin_amdgcn_exp2f(v.x - base);
        sum = fmaf(v.y, c, sum);
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = fmaf(out[(long)s * p.H * DH + e], c, acc[e]);
    }
    sum += lane_xor32(sum);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        acc[e] += lane_xor32(acc[e]);
        if (lane < 32) acc_s[wave][f + e] = acc[e];
    }
    if (lane == 0) sum_s[wave] = sum;
    __syncthreads();
    for (int d = threadIdx.x; d < DH; d += 256) {
        const float s = (sum_s[0] + sum_s[1]) + (sum_s[2] + sum_s[3]);
        const float a = (acc_s[0][d] + acc_s[1][d]) + (acc_s[2][d] + acc_s[3][d]);
        p.ctx[b * p.ldo + (long)h * DH + d] = s == 0.0f ? 0.0f : a / s;
    }
}

constexpr int SPLIT_MIN_ROWS = 256;                 // rows of the smallest chunk

// How many chunks a call is split into (0: one workgroup per request and key head, one launch)
int paged_split_target(int B, int H, int kv_heads, int depth, int type, int max_len) {
    const int n_group = (H / kv_heads + 15) / 16;
    const long units = (long)B * kv_heads * n_group;
    if (max_len <= 512) return 0;
    if (units >= 1024 && max_len <= 2048) return 0;
    const long per = (long)kv_heads * n_group;
    const long t = 1024 / per;
    return (int)(t < 1 ? 1 : t);
}

bool bad_cache(const void* k, const void* v, int64_t s_page, int64_t s_head, int64_t s_row, int type, int depth) {
    const int per16 = type == ESTTS_KV_F32 ? 4 : 8;
    return !k || !v || (reinterpret_cast<uintptr_t>(k) & 15) || (reinterpret_cast<uintptr_t>(v) & 15) || s_page % per16 || s_head % per16 ||
           s_row % per16 || s_row < depth || s_page < 0 || s_head < 0;
}

}  // namespace

extern "C" int estts_page_plan(const estts_page_plan_args* args, void* stream) {
    ESTTS_CHECK_ARG(args != nullptr, "estts_page_plan: null args");
    const estts_page_plan_args& a = *args;
    ESTTS_CHECK_ARG(a.lengths && a.n_new && a.block_table && a.free_pages && a.n_free && a.slots && a.lengths_out && a.n_free_out && a.ws,
                    "estts_page_plan: null pointer");
    ESTTS_CHECK_ARG(a.B > 0 && a.P > 0 && a.n_pages > 0 && a.T > 0 && a.T < (1 << 30) && a.R >= 0 && a.ld_table >= a.P,
                    "estts_page_plan: bad shape");
    ESTTS_CHECK_ARG(a.R == 0 || (int64_t)a.B * a.R == a.T, "estts_page_plan: a padded slot map holds B * R entries");
    ESTTS_CHECK_ARG(a.page > 0 && a.page % 16 == 0, "estts_page_plan: page must be a multiple of 16 (got %d)", a.page);
    ESTTS_CHECK_ARG((int64_t)a.P * a.page < (1LL << 31) && (int64_t)a.n_pages * a.page < (1LL << 31) && (int64_t)a.B * a.P < (1LL << 31),
                    "estts_page_plan: P * page, n_pages * page and B * P must stay below 2^31");
    ESTTS_LAUNCH(page_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, (hipStream_t)stream, a);
    ESTTS_CHECK_LAUNCH("estts_page_plan");
    return 0;
}

extern "C" int estts_page_write(const estts_page_write_args* args, void* stream) {
    ESTTS_CHECK_ARG(args != nullptr, "estts_page_write: null args");
    const estts_page_write_args& a = *args;
    ESTTS_CHECK_ARG(a.k && a.v && a.slots, "estts_page_write: null pointer");
    ESTTS_CHECK_ARG(a.T > 0 && a.heads > 0 && a.depth > 0 && a.n_pages > 0, "estts_page_write: bad shape");
    ESTTS_CHECK_ARG(a.depth % 8 == 0 && a.depth <= 1024 && a.heads <= 65536, "estts_page_write: depth must be a multiple of 8, at most 1024");
    ESTTS_CHECK_ARG(a.page > 0 && a.page % 16 == 0, "estts_page_write: page must be a multiple of 16 (got %d)", a.page);
    ESTTS_CHECK_ARG((int64_t)a.n_pages * a.page < (1LL << 31), "estts_page_write: n_pages * page must stay below 2^31");
    ESTTS_CHECK_ARG(a.type >= ESTTS_KV_F32 && a.type <= ESTTS_KV_F16, "estts_page_write: unknown cache type %d", a.type);
    const int64_t width = (int64_t)a.heads * a.depth;
    ESTTS_CHECK_ARG(!(reinterpret_cast<uintptr_t>(a.k) & 15) && !(reinterpret_cast<uintptr_t>(a.v) & 15) && a.ldk % 4 == 0 && a.ldv % 4 == 0 &&
                    a.ldk >= width && a.ldv >= width, "estts_page_write: rows must be 16-byte aligned and at least heads * depth long");
    ESTTS_CHECK_ARG(!bad_cache(a.k_cache, a.v_cache, a.s_page, a.s_head, a.s_row, a.type, a.depth),
                    "estts_page_write: caches and their strides must be multiples of 16 bytes");
    const int64_t pieces = (int64_t)a.T * (width / 4);
    const int64_t wgs = (pieces + 255) / 256;
    const dim3 grid((unsigned)(wgs < 8192 ? wgs : 8192));
    if (a.type == ESTTS_KV_F32) ESTTS_LAUNCH(page_write_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else if (a.type == ESTTS_KV_BF16) ESTTS_LAUNCH(page_write_kernel<__bf16>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else ESTTS_LAUNCH(page_write_kernel<_Float16>, grid, dim3(256), 0, (hipStream_t)stream, a);
    ESTTS_CHECK_LAUNCH("estts_page_write");
    return 0;
}

extern "C" int64_t estts_paged_attention_ws_bytes(int32_t B, int32_t H, int32_t kv_heads, int32_t depth, int32_t type, int32_t max_len) {
    if (B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads || depth <= 0 || max_len <= 0) return 0;      // (estts_paged_attention says why not)
    const int target = paged_split_target(B, H, kv_heads, depth, type, max_len);
    return target ? PagedScratch::bytes((long)target + B, H, depth, B) : 0;
}

template <typename T, int DH>
static void launch_paged_attention(const estts_paged_attention_args& a, int target, hipStream_t stream) {
    const int n_items = target ? target + a.B : a.B, n_group = (a.H / a.kv_heads + 15) / 16;
    const int units = n_items * a.kv_heads;
    const dim3 grid(n_group > 1 ? (units + 7) / 8 * 8 * n_group : units);
    if (a.key_mask) ESTTS_LAUNCH((paged_attention_kernel<T, DH, true>), grid, dim3(ATT_WAVES * 64), 0, stream, a, target, SPLIT_MIN_ROWS);
    else ESTTS_LAUNCH((paged_attention_kernel<T, DH, false>), grid, dim3(ATT_WAVES * 64), 0, stream, a, target, SPLIT_MIN_ROWS);
    if (target) ESTTS_LAUNCH(paged_join_kernel<DH>, dim3(a.H, a.B), dim3(256), 0, stream, a, n_items);
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
    ESTTS_CHECK_ARG((int64_t)a.B * a.max_len < (1LL << 38) && ((int64_t)a.B + 1024) * a.H < (1LL << 28),
                    "estts_paged_attention: B * max_len must stay below 2^38 and B * H below 2^28");
    const int target = paged_split_target(a.B, a.H, a.kv_heads, a.depth, a.type, a.max_len);
    const int64_t need = target ? PagedScratch::bytes((long)target + a.B, a.H, a.depth, a.B) : 0;
    ESTTS_CHECK_ARG(need == 0 || (a.ws && a.ws_bytes >= need && !(reinterpret_cast<uintptr_t>(a.ws) & 15)),
                    "estts_paged_attention: this call needs %ld bytes of scratch, 16-byte aligned (given: %ld)", (long)need, (long)a.ws_bytes);
    if (a.type == ESTTS_KV_F32) launch_paged_attention<float>(a, target, (hipStream_t)stream);
    else if (a.type == ESTTS_KV_BF16) launch_paged_attention<__bf16>(a, target, (hipStream_t)stream);
    else launch_paged_attention<_Float16>(a, target, (hipStream_t)stream);
    ESTTS_CHECK_LAUNCH("estts_paged_attention");
    return 0;
}
