// page_bounds.cu — per-page channel bounds of the keys, and the choice of the pages a query attends to.
//
// Bounds of a (layer, page, KV head): the largest and the smallest key value of every channel, rounded outwards to 8-bit
// whole numbers of 2^e, e = smallest integer with max|k| <= 127 * 2^e:  b_max = ceil(max / 2^e), b_min = floor(min / 2^e).
// ceil(ceil(x) / 2^i) = ceil(x / 2^i), so widening page bounds key by key gives the bytes a single pass would.
// Score of a page for a group of query heads: q8 = rint(q / 2^f), f = smallest integer with max|q| <= 127 * 2^f, and
//   score = max over heads of 2^(e + f) * sum_d (q8_d > 0 ? q8_d * b_max_d : q8_d * b_min_d),
// an upper bound of q8 . k over the page's keys.  The sum is one of whole numbers below 2^22: it is the same in every
// order and on every unit, so equal scores are equal bits and the selection is reproducible (ties: lowest page).
// As a contraction: [q8 clipped to >= 0, q8 clipped to <= 0] . [b_max, b_min], 2 D long, on int8 mma.sync tiles.
//
// The score pass reads (2 D + 1) bytes per page and KV head, D + 1/2 times fewer than 2 P rows of 16 bits would be: HBM-
// bound for long contexts; the selection runs on the scores in shared memory, one CTA per (sequence, KV head).
#include <atomic>

#include "kernels.hpp"
#include "kv_common.cuh"

namespace drkv {

namespace {

constexpr uint32_t FULL = 0xffffffffu;
constexpr uint32_t kKeyHole = 0, kKeyForced = 0xffffffffu;

// Smallest e with |x| <= 127 * 2^e (127 = 1.984375 * 2^6), within -126 .. 121; |x| by its fp32 bits, infinity included.
__device__ __forceinline__ int bound_exponent(uint32_t abs_bits) {
    const int e = (int)(abs_bits >> 23) - 127 - 6 + ((abs_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return max(-126, min(121, e));
}

// D / 32 consecutive channels of one stored key row, as fp32.
template <bool POOL8, typename T, int D>
__device__ __forceinline__ void load_key(const uint8_t* block, const BoundsParams& p, int head, int slot, int lane, float (&x)[D / 32]) {
    constexpr int C = D / 32;
    const int64_t row = (int64_t)head * p.page_size + slot;
    if (POOL8) {
        const float scale = exp2_int((int)block[2 * p.plane_bytes + row] - 127);
        const uint16_t* src = reinterpret_cast<const uint16_t*>(block + row * D + lane * C);
#pragma unroll
        for (int i = 0; i < C / 2; i++) {
            const float2 f = Elem<__half>::unpack2(e4m3x2_to_f16x2(src[i]));
            x[2 * i] = f.x * scale;
            x[2 * i + 1] = f.y * scale;
        }
    } else {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(block + (row * D + lane * C) * 2);
#pragma unroll
        for (int i = 0; i < C / 2; i++) {
            const float2 f = Elem<T>::unpack2(src[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

// One warp per (page, KV head).  What a launch covers:
//   rows != null    the page of every batch entry's position, that slot (entries of one sequence in the same page are
//                   gathered by the first of them: one writer per page)
//   table != null   the pages of one sequence that hold tokens [pos_start, pos_start + m), those slots
//   neither         pages [page0, page0 + n_items), every slot
// A page whose slot 0 is covered starts anew, any other is widened.
template <bool POOL8, typename T, int D>
__global__ void __launch_bounds__(256) bounds_kernel(const BoundsParams p) {
    constexpr int C = D / 32;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t wid = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int item = (int)(wid / p.num_kv_heads), head = (int)(wid - (int64_t)item * p.num_kv_heads);
    if (item >= p.n_items) return;
    const int layer = p.layer + blockIdx.y;
    const int P = p.page_size;
    int page = -1, slot_lo = 0, slot_hi = P, row = 0, logical = 0;
    bool fresh = true;
    if (p.rows != nullptr) {
        row = __ldg(p.rows + item);
        const int pos = __ldg(p.pos + item) + p.pos_offset;
        if (pos < 0 || row < 0 || row >= p.max_rows) return;
        logical = pos / P;
        if (logical >= p.table_stride) return;
        for (int j0 = 0; j0 < item; j0 += 32) {                             // an earlier entry in the same page does it all
            const int j = j0 + lane;
            const bool same = j < item && __ldg(p.rows + j) == row && __ldg(p.pos + j) + p.pos_offset >= 0 &&
                              (__ldg(p.pos + j) + p.pos_offset) / P == logical;
            if (__any_sync(FULL, same)) return;
        }
        page = __ldg(p.tables + (int64_t)row * p.table_stride + logical);
        slot_lo = pos - logical * P;
        slot_hi = slot_lo + 1;
        fresh = slot_lo == 0;
    } else if (p.tables != nullptr) {
        logical = p.pos_start / P + item;
        if (logical >= p.table_stride) return;
        page = __ldg(p.tables + (int64_t)p.row * p.table_stride + logical);
        const int64_t first = (int64_t)logical * P;
        slot_lo = p.pos_start > first ? (int)(p.pos_start - first) : 0;
        const int64_t end = (int64_t)p.pos_start + p.m - first;
        slot_hi = end < P ? (int)end : P;
        fresh = slot_lo == 0;
    } else {
        page = p.page0 + item;
    }
    if (page < 0 || page >= p.max_pages) return;
    const uint8_t* block = p.pool + layer * p.layer_bytes + (int64_t)page * p.block_bytes;
    const int64_t at = ((int64_t)layer * p.max_pages + page) * p.num_kv_heads + head;
    int8_t* bounds = p.bounds + at * 2 * D;

    float hi[C], lo[C];
#pragma unroll
    for (int i = 0; i < C; i++) {
        hi[i] = -INFINITY;
        lo[i] = INFINITY;
    }
    auto take = [&](int slot) {
        float x[C];
        load_key<POOL8, T, D>(block, p, head, slot, lane, x);
#pragma unroll
        for (int i = 0; i < C; i++) {                                       // NaN is ignored
            hi[i] = fmaxf(hi[i], x[i]);
            lo[i] = fminf(lo[i], x[i]);
        }
    };
#pragma unroll 4
    for (int s = slot_lo; s < slot_hi; s++) take(s);
    if (p.rows != nullptr) {                                                // later entries in the same page
        for (int j0 = item + 1; j0 < p.n_items; j0 += 32) {
            const int j = j0 + lane;
            int slot = -1;
            if (j < p.n_items && __ldg(p.rows + j) == row) {
                const int pos = __ldg(p.pos + j) + p.pos_offset;
                if (pos >= 0 && pos / P == logical) slot = pos - logical * P;
            }
            for (uint32_t left = __ballot_sync(FULL, slot >= 0); left; left &= left - 1) {
                const int s = __shfl_sync(FULL, slot, __ffs(left) - 1);
                take(s);
                fresh |= s == 0;
            }
        }
    }
    if (!fresh) {
        const float unit = exp2_int(p.exponents[at]);
#pragma unroll
        for (int i = 0; i < C; i++) {
            hi[i] = fmaxf(hi[i], bounds[lane * C + i] * unit);
            lo[i] = fminf(lo[i], bounds[D + lane * C + i] * unit);
        }
    }
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < C; i++) {
        if (hi[i] < lo[i]) hi[i] = lo[i] = 0.f;                             // nothing but NaN
        amax = max(amax, max(__float_as_uint(hi[i]) & 0x7fffffffu, __float_as_uint(lo[i]) & 0x7fffffffu));
    }
    const int e = bound_exponent(__reduce_max_sync(FULL, amax));
    const float inv = exp2_int(-e);
#pragma unroll
    for (int i = 0; i < C; i++) {
        float a = ceilf(hi[i] * inv), b = floorf(lo[i] * inv);
        if (hi[i] > 0.f) a = fmaxf(a, 1.f);                                 // the product may have underflowed
        if (lo[i] < 0.f) b = fminf(b, -1.f);
        bounds[lane * C + i] = (int8_t)fmaxf(-127.f, fminf(127.f, a));
        bounds[D + lane * C + i] = (int8_t)fmaxf(-127.f, fminf(127.f, b));
    }
    if (lane == 0) p.exponents[at] = (int8_t)e;
}

// The bounds of a page follow it when it is copied on write.
__global__ void __launch_bounds__(256) bounds_copy_kernel(const BoundsParams p, int head_dim, int src_page, int dst_page) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t per = (int64_t)p.num_kv_heads * 2 * head_dim;
    const int64_t src = ((int64_t)blockIdx.x * p.max_pages + src_page), dst = ((int64_t)blockIdx.x * p.max_pages + dst_page);
    for (int64_t i = threadIdx.x; i < per / 16; i += blockDim.x) stg16(p.bounds + dst * per + 16 * i, ldg16(p.bounds + src * per + 16 * i));
    for (int i = threadIdx.x; i < p.num_kv_heads; i += blockDim.x)
        p.exponents[dst * p.num_kv_heads + i] = p.exponents[src * p.num_kv_heads + i];
}

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// fp32 order as unsigned order; finite or infinite scores fall in 1 .. 0xfffffffe
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);                            // -0 counts as 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One warp per 8 pages at a time of one (sequence, KV head): the pages are the columns of the int8 tiles, the group's heads
// the rows.  A lane takes whole 16-byte chunks of a page's 2 D bound bytes (contraction order is free) straight from
// global memory into operand registers; the query bytes stay in registers over all pages of the warp.
// grid (page blocks, KV heads, sequences); keys[(seq * Hkv + head) * stride + page].
constexpr int kScoreWarps = 4;
template <typename T, int D, bool HI>
__global__ void __launch_bounds__(kScoreWarps * 32) page_score_kernel(const SelectParams p, int pages_per_cta) {
    constexpr int CH = D / 64;                                              // query chunks (16 dims) a lane owns
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int row = __ldg(p.rows + b);
    const int len = min(__ldg(p.kv_len + b), p.max_kv_len);
    if (len <= 0 || row < 0 || row >= p.max_rows) return;
    const int n = min((len - 1) / p.page_size + 1, p.table_stride);
    const int first = blockIdx.x * pages_per_cta, last = min(n, first + pages_per_cta);
    if (first >= last) return;
    // ---- query bytes ----
    uint32_t up[HI ? 2 : 1][CH][4], down[HI ? 2 : 1][CH][4];
    int f[HI ? 2 : 1];
#pragma unroll
    for (int r = 0; r < (HI ? 2 : 1); r++) {
        const int head = g + 8 * r;
        const bool live = head < p.group;
        const T* q = reinterpret_cast<const T*>(p.q) + (((int64_t)b * p.num_kv_heads + h) * p.group + head) * D;
        float x[CH][16];
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                Vec16 v = Vec16{{0u, 0u, 0u, 0u}};
                if (live) v = ldg16(q + 16 * (t + 4 * i) + 8 * c);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 y = Elem<T>::unpack2(v.w[j]);
                    x[i][8 * c + 2 * j] = y.x;
                    x[i][8 * c + 2 * j + 1] = y.y;
                    // NaN counts as nothing, here and below
                    amax = max(amax, y.x == y.x ? __float_as_uint(y.x) & 0x7fffffffu : 0u);
                    amax = max(amax, y.y == y.y ? __float_as_uint(y.y) & 0x7fffffffu : 0u);
                }
            }
        amax = max(amax, __shfl_xor_sync(FULL, amax, 1));
        amax = max(amax, __shfl_xor_sync(FULL, amax, 2));
        f[r] = bound_exponent(amax);
        const float inv = exp2_int(-f[r]);
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t u = 0, d = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float y = x[i][4 * k + j];
                    const int v = y == y ? max(-127, min(127, __float2int_rn(fmaxf(-128.f, fminf(128.f, y * inv))))) : 0;
                    u |= (uint32_t)(max(v, 0) & 0xff) << (8 * j);
                    d |= (uint32_t)(min(v, 0) & 0xff) << (8 * j);
                }
                up[r][i][k] = u;
                down[r][i][k] = d;
            }
    }
    const int32_t* table = p.tables + (int64_t)row * p.table_stride;
    uint32_t* keys = p.keys + ((int64_t)b * p.num_kv_heads + h) * p.key_stride;
    const int64_t layer0 = (int64_t)p.layer * p.max_pages;
#pragma unroll 2
    for (int p0 = first + 8 * w; p0 < last; p0 += 8 * kScoreWarps) {
        // lane's page is p0 + g; the bounds of a hole are not read
        int page = -1;
        if (p0 + g < last) page = __ldg(table + p0 + g);
        if (page >= p.max_pages) {
            atomicExch(p.error_word, (int)KERR_BAD_PAGE);
            page = -1;
        }
        const int64_t at = (layer0 + (page < 0 ? 0 : page)) * p.num_kv_heads + h;
        const int8_t* bounds = p.bounds + at * 2 * D;
        Vec16 v[2 * CH];
#pragma unroll
        for (int i = 0; i < 2 * CH; i++) {
            v[i] = Vec16{{0u, 0u, 0u, 0u}};
            if (page >= 0) v[i] = ldg16(bounds + 16 * (t + 4 * i));
        }
        const int e_own = page >= 0 ? p.exponents[at] : 0;
        int acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                mma_s8(acc, up[0][i][k], HI ? up[HI ? 1 : 0][i][k] : 0u, up[0][i][k + 1], HI ? up[HI ? 1 : 0][i][k + 1] : 0u,
                       v[i].w[k], v[i].w[k + 1]);
                mma_s8(acc, down[0][i][k], HI ? down[HI ? 1 : 0][i][k] : 0u, down[0][i][k + 1], HI ? down[HI ? 1 : 0][i][k + 1] : 0u,
                       v[CH + i].w[k], v[CH + i].w[k + 1]);
            }
        // heads g (and g + 8), pages p0 + 2t and p0 + 2t + 1
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int e = __shfl_sync(FULL, e_own, 4 * (2 * t + c));
            float best = -INFINITY;
#pragma unroll
            for (int r = 0; r < (HI ? 2 : 1); r++) {
                const int ef = e + f[r], e1 = max(-126, min(127, ef));
                const float s = (float)acc[2 * r + c] * exp2_int(e1) * exp2_int(ef - e1);
                if (g + 8 * r < p.group) best = fmaxf(best, s);
            }
            best = fmaxf(best, __shfl_xor_sync(FULL, best, 4));
            best = fmaxf(best, __shfl_xor_sync(FULL, best, 8));
            best = fmaxf(best, __shfl_xor_sync(FULL, best, 16));
            const int pg = __shfl_sync(FULL, page, 4 * (2 * t + c)), idx = p0 + 2 * t + c;
            if (g == 0 && idx < last)
                keys[idx] = pg < 0 ? kKeyHole : (idx < p.first_pages || idx >= n - p.last_pages) ? kKeyForced : ordered(best);
        }
    }
}

// One CTA per (KV head, sequence): the top_pages largest keys (ties: lowest page), pages ascending, -1 behind them.
// The k-th largest key is found bit by bit from the top: how many keys reach the candidate decides the bit.
constexpr int kSelectThreads = 512;
__global__ void __launch_bounds__(kSelectThreads) page_select_kernel(const SelectParams p, int smem_keys) {
    extern __shared__ uint32_t s_keys[];
    __shared__ int2 s_warp[kSelectThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int64_t pair = (int64_t)b * p.num_kv_heads + h;
    const int row = __ldg(p.rows + b);
    const int len = min(__ldg(p.kv_len + b), p.max_kv_len);
    const int n = len <= 0 || row < 0 || row >= p.max_rows ? 0 : min((len - 1) / p.page_size + 1, p.table_stride);
    const uint32_t* keys = p.keys + pair * p.key_stride;
    int32_t* sel = p.sel + pair * p.top_pages;
    int mine = 0;
    for (int i = tid; i < n; i += kSelectThreads) {
        const uint32_t k = keys[i];
        if (i < smem_keys) s_keys[i] = k;
        mine += k != kKeyHole;
    }
    auto key_at = [&](int i) { return i < smem_keys ? s_keys[i] : keys[i]; };
    auto block_sum = [&](int v) -> int {
        v = __reduce_add_sync(FULL, v);
        __syncthreads();
        if (lane == 0) s_warp[w].x = v;
        __syncthreads();
        int s = 0;
#pragma unroll
        for (int i = 0; i < kSelectThreads / 32; i++) s += s_warp[i].x;
        return s;
    };
    const int resident = block_sum(mine);
    const int k = min(p.top_pages, resident);
    uint32_t cut = 1;                                                       // everything resident
    int above = 0;                                                          // keys > cut
    if (resident > k) {
        cut = 0;
        int reach = resident;                                               // keys >= cut, cut's lower bits being 0
        for (int bit = 31; bit >= 0 && reach > k; bit--) {
            const uint32_t cand = cut | (1u << bit);
            int c = 0;
            for (int i = tid; i < n; i += kSelectThreads) c += key_at(i) >= cand;
            c = block_sum(c);
            if (c >= k) {
                cut = cand;
                reach = c;
            }
        }
        int c = 0;
        for (int i = tid; i < n; i += kSelectThreads) c += key_at(i) > cut;
        above = block_sum(c);
        if (reach == k) above = -1;                                         // exactly k keys reach the cut: no ties to break
    }
    const int ties = above < 0 || resident == k ? n : k - above;            // keys equal to the cut that are taken, lowest first
    const bool all = above < 0 || resident == k;
    int done = 0, tied = 0;
    for (int base = 0; base < n; base += kSelectThreads) {
        const int i = base + tid;
        const uint32_t key = i < n ? key_at(i) : kKeyHole;
        const bool eq = !all && key == cut && key != kKeyHole;
        const bool gt = key != kKeyHole && (all ? key >= cut : key > cut);
        const uint32_t beq = __ballot_sync(FULL, eq), bgt = __ballot_sync(FULL, gt);
        __syncthreads();
        if (lane == 0) s_warp[w] = make_int2(__popc(bgt), __popc(beq));
        __syncthreads();
        int gt_before = done, eq_before = tied;
#pragma unroll
        for (int v = 0; v < kSelectThreads / 32; v++) {
            if (v < w) {
                gt_before += s_warp[v].x;
                eq_before += s_warp[v].y;
            }
            done += s_warp[v].x;
            tied += s_warp[v].y;
        }
        const uint32_t below = (1u << lane) - 1;
        gt_before += __popc(bgt & below);
        eq_before += __popc(beq & below);
        const int at = gt_before + min(eq_before, ties);
        if ((gt || (eq && eq_before < ties)) && at < k) sel[at] = i;
    }
    for (int i = k + tid; i < p.top_pages; i += kSelectThreads) sel[i] = -1;
}

template <bool POOL8, typename T>
cudaError_t launch_bounds_d(const BoundsParams& p, int head_dim, dim3 grid, cudaStream_t s) {
    switch (head_dim) {
        case 64: return launch_pdl(bounds_kernel<POOL8, T, 64>, grid, dim3(256), 0, s, p);
        case 128: return launch_pdl(bounds_kernel<POOL8, T, 128>, grid, dim3(256), 0, s, p);
        case 256: return launch_pdl(bounds_kernel<POOL8, T, 256>, grid, dim3(256), 0, s, p);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T, int D>
cudaError_t launch_score(const SelectParams& p, int num_sms, cudaStream_t s) {
    const int pages = min((p.max_kv_len - 1) / p.page_size + 1, p.table_stride);
    // a CTA takes 8 pages a warp at a time; more per CTA (the query bytes are made once) while 8 CTAs an SM remain
    int per_cta = 8 * kScoreWarps;
    while (per_cta < 1024 && (int64_t)((pages + 2 * per_cta - 1) / (2 * per_cta)) * p.num_kv_heads * p.n_seq >= 8 * num_sms) per_cta *= 2;
    const dim3 grid((pages + per_cta - 1) / per_cta, p.num_kv_heads, p.n_seq);
    return p.group > 8 ? launch_pdl(page_score_kernel<T, D, true>, grid, dim3(kScoreWarps * 32), 0, s, p, per_cta)
                       : launch_pdl(page_score_kernel<T, D, false>, grid, dim3(kScoreWarps * 32), 0, s, p, per_cta);
}

}  // namespace

cudaError_t launch_bounds(const BoundsParams& p, bool pool8, int head_dim, int dtype, int num_layers, cudaStream_t stream) {
    if (p.n_items <= 0 || num_layers <= 0) return cudaSuccess;
    const int64_t blocks = ((int64_t)p.n_items * p.num_kv_heads + 7) / 8;
    if (blocks > 0x7fffffff || num_layers > 65535) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)blocks, num_layers);
    if (pool8) return launch_bounds_d<true, __half>(p, head_dim, grid, stream);
    return dtype == DRKV_DTYPE_F16 ? launch_bounds_d<false, __half>(p, head_dim, grid, stream)
                                   : launch_bounds_d<false, __nv_bfloat16>(p, head_dim, grid, stream);
}

cudaError_t launch_bounds_copy(const BoundsParams& p, int head_dim, int src_page, int dst_page, int num_layers, cudaStream_t stream) {
    return launch_pdl(bounds_copy_kernel, dim3(num_layers), dim3(256), 0, stream, p, head_dim, src_page, dst_page);
}

cudaError_t launch_select_pages(const SelectParams& p, int head_dim, int dtype, int num_sms, cudaStream_t stream) {
    if (p.n_seq <= 0) return cudaSuccess;
    if (p.n_seq > 65535 || p.num_kv_heads > 65535 || p.group < 1 || p.group > 16) return cudaErrorInvalidValue;
    const bool f16 = dtype == DRKV_DTYPE_F16;
    cudaError_t e = cudaSuccess;
    if (p.max_kv_len > 0) {
        switch (head_dim) {
            case 64: e = f16 ? launch_score<__half, 64>(p, num_sms, stream) : launch_score<__nv_bfloat16, 64>(p, num_sms, stream); break;
            case 128: e = f16 ? launch_score<__half, 128>(p, num_sms, stream) : launch_score<__nv_bfloat16, 128>(p, num_sms, stream); break;
            case 256: e = f16 ? launch_score<__half, 256>(p, num_sms, stream) : launch_score<__nv_bfloat16, 256>(p, num_sms, stream); break;
            default: return cudaErrorInvalidValue;
        }
        if (e != cudaSuccess) return e;
    }
    // keys beyond 12 288 (48 KB) of a sequence are read from global memory (L2) in every round
    const int pages = p.max_kv_len > 0 ? min((p.max_kv_len - 1) / p.page_size + 1, p.table_stride) : 0;
    const int smem_keys = pages < 12288 - 256 ? pages : 12288 - 256;
    return launch_pdl(page_select_kernel, dim3(p.num_kv_heads, p.n_seq), dim3(kSelectThreads), (size_t)smem_keys * 4, stream, p, smem_keys);
}

}  // namespace drkv
