// Paged key / value memory: the page plan of a step, the write of new rows into the pages, the attention of one new row per
// request over its pages (see estts_page_plan, estts_page_write, estts_paged_attention in include/estts.h).
#include "common.h"

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
// A workgroup owns one (request, query head).  Sixteen lanes share a key row; each of the sixteen groups sweeps every sixteenth
// key with its own running maximum, sum and output, which meet in LDS at the end.
template <typename T, int DH>
__global__ __launch_bounds__(256) void paged_attention_kernel(const estts_paged_attention_args p) {
    constexpr int PER = DH / 16;
    __shared__ float o_s[16][DH], m_s[16], l_s[16];
    const int h = blockIdx.x, b = blockIdx.y;
    const int grp = threadIdx.x >> 4, i = threadIdx.x & 15;
    const int hk = h / (p.H / p.kv_heads);
    const int len = min(min(max(p.lengths[b], 0), p.P * p.page), p.max_len);
    const int* table = p.block_table + b * p.ld_table;
    const T* kc = static_cast<const T*>(p.k_cache) + hk * p.s_head + i * PER;
    const T* vc = static_cast<const T*>(p.v_cache) + hk * p.s_head + i * PER;
    float q[PER], o[PER] = {};
    for (int e = 0; e < PER; ++e) q[e] = p.q[b * p.ldq + h * DH + i * PER + e] * (p.scale * 1.4426950408889634f);
    float m = -INFINITY, l = 0.0f;
    for (int j = grp; j < len; j += 16) {
        const int id = table[j / p.page];
        if (id < 0 || id >= p.n_pages) continue;
        if (p.key_mask && p.key_mask[b * p.mask_sb + j * p.mask_ss] != 0.0f) continue;
        const long at = id * p.s_page + (long)(j % p.page) * p.s_row;
        float s = 0.0f;
        for (int e = 0; e < PER; ++e) s = fmaf(q[e], (float)kc[at + e], s);
        for (int d = 1; d < 16; d <<= 1) s += __shfl_xor(s, d);
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.0f : top;
        const float c = exp2f(m - base), w = exp2f(s - base);
        l = l * c + w;
        for (int e = 0; e < PER; ++e) o[e] = fmaf(w, (float)vc[at + e], o[e] * c);
        m = top;
    }
    for (int e = 0; e < PER; ++e) o_s[grp][i * PER + e] = o[e];
    if (i == 0) { m_s[grp] = m; l_s[grp] = l; }
    __syncthreads();
    for (int d = threadIdx.x; d < DH; d += 256) {
        float top = -INFINITY, sum = 0.0f, acc = 0.0f;
        for (int g = 0; g < 16; ++g) top = fmaxf(top, m_s[g]);
        const float base = top == -INFINITY ? 0.0f : top;
        for (int g = 0; g < 16; ++g) {
            const float c = exp2f(m_s[g] - base);
            sum += l_s[g] * c;
            acc = fmaf(o_s[g][d], c, acc);
        }
        p.ctx[b * p.ldo + h * DH + d] = sum == 0.0f ? 0.0f : acc / sum;
    }
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
    return 0;
}

template <typename T>
static void launch_paged_attention(const estts_paged_attention_args& a, hipStream_t stream) {
    const dim3 grid(a.H, a.B);
    if (a.depth == 32) ESTTS_LAUNCH((paged_attention_kernel<T, 32>), grid, dim3(256), 0, stream, a);
    else if (a.depth == 64) ESTTS_LAUNCH((paged_attention_kernel<T, 64>), grid, dim3(256), 0, stream, a);
    else ESTTS_LAUNCH((paged_attention_kernel<T, 128>), grid, dim3(256), 0, stream, a);
}

extern "C" int estts_paged_attention(const estts_paged_attention_args* args, void* stream) {
    ESTTS_CHECK_ARG(args != nullptr, "estts_paged_attention: null args");
    estts_paged_attention_args a = *args;
    ESTTS_CHECK_ARG(a.q && a.block_table && a.lengths && a.ctx, "estts_paged_attention: null pointer");
    ESTTS_CHECK_ARG(a.B > 0 && a.B <= 65535 && a.H > 0 && a.kv_heads > 0 && a.H % a.kv_heads == 0 && a.P > 0 && a.n_pages > 0 && a.ld_table >= a.P,
                    "estts_paged_attention: bad shape (B 1 .. 65535, heads a multiple of kv_heads)");
    ESTTS_CHECK_ARG(a.depth == 32 || a.depth == 64 || a.depth == 128, "estts_paged_attention: depth must be 32, 64 or 128 (got %d)", a.depth);
    ESTTS_CHECK_ARG(a.page > 0 && a.page % 16 == 0, "estts_paged_attention: page must be a multiple of 16 (got %d)", a.page);
    ESTTS_CHECK_ARG((int64_t)a.P * a.page < (1LL << 31) && (int64_t)a.n_pages * a.page < (1LL << 31),
                    "estts_paged_attention: P * page and n_pages * page must stay below 2^31");
    ESTTS_CHECK_ARG(a.type >= ESTTS_KV_F32 && a.type <= ESTTS_KV_F16, "estts_paged_attention: unknown cache type %d", a.type);
    const int64_t width = (int64_t)a.H * a.depth;
    ESTTS_CHECK_ARG(!(reinterpret_cast<uintptr_t>(a.q) & 15) && a.ldq % 4 == 0 && a.ldq >= width && a.ldo >= width,
                    "estts_paged_attention: query rows must be 16-byte aligned, rows at least H * depth long");
    ESTTS_CHECK_ARG(!bad_cache(a.k_cache, a.v_cache, a.s_page, a.s_head, a.s_row, a.type, a.depth),
                    "estts_paged_attention: caches and their strides must be multiples of 16 bytes");
    ESTTS_CHECK_ARG(a.s_row * (int64_t)a.page < (1LL << 28), "estts_paged_attention: the rows of one page must span less than 2^28 elements");
    ESTTS_CHECK_ARG(a.max_len >= 0, "estts_paged_attention: max_len must not be negative");
    if (a.max_len == 0 || (int64_t)a.max_len > (int64_t)a.P * a.page) a.max_len = a.P * a.page;
    if (a.type == ESTTS_KV_F32) launch_paged_attention<float>(a, (hipStream_t)stream);
    else if (a.type == ESTTS_KV_BF16) launch_paged_attention<__bf16>(a, (hipStream_t)stream);
    else launch_paged_attention<_Float16>(a, (hipStream_t)stream);
    ESTTS_CHECK_LAUNCH("estts_paged_attention");
    return 0;
}
