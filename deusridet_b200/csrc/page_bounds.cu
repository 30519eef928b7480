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
// The score pass reads 2 D + 1 bytes per page and KV head where the page's K and V rows are 4 P D in 16 bits.  86 MB take it
// 20 us, 4.3 TB/s with DRAM 46 % and the issue slots 48 % busy: bound by the latency of a warp's 32 to 64 pages, two to four
// stages behind the making of its query bytes.  The selection runs on the scores in shared memory, one CTA per (sequence, KV
// head): a chain of scans, latency too.
#include <atomic>

#include "kernels.hpp"
#include "kv_common.cuh"
#include "row_tiles.cuh"
#include "sm100_primitives.cuh"

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

// One warp per (page, KV head), or a CTA whose warps share the slots (SPLIT: what covers more than a token a page and has too
// few pages to fill the SMs with a warp each; 2 048 of 8 heads of 256 on pages of 128: 9 us, by one warp each 63).  What a launch covers:
//   rows != null    the page of every batch entry's position, that slot (entries of one sequence in the same page are
//                   gathered by the first of them: one writer per page)
//   table != null   the pages of one sequence that hold tokens [pos_start, pos_start + m), those slots
//   neither         pages [page0, page0 + n_items), every slot
// A page whose slot 0 is covered starts anew, any other is widened.
template <bool POOL8, typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(256) bounds_kernel(const BoundsParams p) {
    constexpr int C = D / 32, WARPS = SPLIT ? 8 : 1;
    __shared__ float s_hi[SPLIT ? 8 : 1][D], s_lo[SPLIT ? 8 : 1][D];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int w = threadIdx.x >> 5;
    const int64_t wid = SPLIT ? blockIdx.x : (int64_t)blockIdx.x * 8 + w;
    const int item = (int)(wid / p.num_kv_heads), head = (int)(wid - (int64_t)item * p.num_kv_heads);
    if (item >= p.n_items) return;
    const int layer = p.layer + blockIdx.y;
    const int P = p.page_size;
    int page = -1, slot_lo = 0, slot_hi = P, row = 0, logical = 0;
    bool fresh = true;
    if (!SPLIT && p.rows != nullptr) {
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
    for (int s = slot_lo + (SPLIT ? w : 0); s < slot_hi; s += WARPS) take(s);
    if (!SPLIT && p.rows != nullptr) {                                                // later entries in the same page
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
    if (SPLIT) {
#pragma unroll
        for (int i = 0; i < C; i++) {
            s_hi[w][lane + 32 * i] = hi[i];                                 // channel lane * C + i
            s_lo[w][lane + 32 * i] = lo[i];
        }
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int v = 1; v < WARPS; v++)
#pragma unroll
            for (int i = 0; i < C; i++) {
                hi[i] = fmaxf(hi[i], s_hi[v][lane + 32 * i]);
                lo[i] = fminf(lo[i], s_lo[v][lane + 32 * i]);
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

// One warp walks pages of one (sequence, KV head), 16 to an int8 tile: the pages are its rows, the group's heads its columns
// (8 a tile), so that the maximum over the heads is two shuffles.  Contraction order is free: a lane takes whole 16-byte
// chunks of a page's 2 D bound bytes, and the query bytes of the same dims stay in registers over all pages.  Bounds come by
// cp.async into a ring per warp, 4 KB a stage at head_dim 128, three stages ahead.  42 000 pages of 8 heads (86 MB) take
// 20 us; with heads as rows, their scales applied per page, and bounds held in registers 27 to 33 us.
// The warps of a CTA take neighbouring heads of the same pages (their bounds lie side by side in memory), and where there
// are fewer than four, stretches of the pages.  grid (page blocks, KV heads / heads_per_cta, sequences);
// keys[(seq * Hkv + head) * stride + page].
constexpr int kScoreWarps = 4, kScorePages = 16;                            // pages of a stage
template <int D> constexpr int kScoreStages = D == 256 ? 3 : 4;
template <typename T, int D, bool HI>
__global__ void __launch_bounds__(kScoreWarps * 32) page_score_kernel(const SelectParams p, int pages_per_cta, int heads_per_cta) {
    constexpr int CH = D / 64;                                              // query chunks (16 dims) a lane owns
    constexpr int ROWB = 2 * D, CPR = ROWB / 16, STAGE = kScorePages * ROWB, STAGES = kScoreStages<D>;
    constexpr int NR = HI ? 2 : 1;
    extern __shared__ __align__(128) uint8_t smem[];
    const int b = blockIdx.z, lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y * heads_per_cta + w % heads_per_cta, part = w / heads_per_cta, parts = kScoreWarps / heads_per_cta;
    // lengths, rows and tables come from further back than the kernel directly in front
    const int row = __ldg(p.rows + b);
    const int len = min(__ldg(p.kv_len + b), p.max_kv_len);
    const int n = len <= 0 || row < 0 || row >= p.max_rows ? 0 : min((len - 1) / p.page_size + 1, p.table_stride);
    const int per_part = pages_per_cta / parts;                             // a multiple of 32
    const int begin = blockIdx.x * pages_per_cta + part * per_part, last = min(n, begin + per_part);
    const int32_t* table = p.tables + (int64_t)row * p.table_stride;
    auto page_ids = [&](int i) -> int {                                     // lane i: page i of a window of 32
        return i + lane < last ? __ldg(table + i + lane) : -1;
    };
    int iss32 = -1, iss_next = -1;
    if (begin < last) {
        iss32 = page_ids(begin);
        iss_next = page_ids(begin + 32);
    }
    pdl_wait();
    pdl_launch_dependents();
    if (begin >= last) return;
    const int64_t layer0 = (int64_t)p.layer * p.max_pages;
    auto checked = [&](int page) -> int {
        if (page >= p.max_pages) {
            atomicExch(p.error_word, (int)KERR_BAD_PAGE);
            return -1;
        }
        return page;
    };
    // (a plain load: the kernel in front may have written them while this one was already running)
    auto exponent_of = [&](int page) -> int { return page >= 0 ? p.exponents[(layer0 + page) * p.num_kv_heads + h] : 0; };
    iss32 = checked(iss32);
    iss_next = checked(iss_next);
    int page32 = iss32, next32 = iss_next;                                  // of the window being scored, and the one behind it
    int e32 = exponent_of(page32), next_e = exponent_of(next32);
    const uint32_t ring = smem_u32(smem) + w * STAGES * STAGE;
    const int n_stages = (last - begin + kScorePages - 1) / kScorePages;
    // a lane's chunks of a stage are 32 apart: c = lane + 32 j, page c / CPR of the stage (see tile_off)
    const int8_t* lane_src = p.bounds + (layer0 * p.num_kv_heads + h) * ROWB + 16 * (lane % CPR);
    const uint32_t lane_dst = tile_off<ROWB>(lane / CPR, lane % CPR), page_bytes = (uint32_t)p.num_kv_heads * ROWB;
    auto issue = [&](int s) {
        if ((s & 1) == 0 && s > 0) {
            iss32 = iss_next;
            iss_next = checked(page_ids(begin + s * kScorePages + 32));
        }
        const uint32_t stage = ring + (s % STAGES) * STAGE;
#pragma unroll
        for (int j = 0; j < CPR / 2; j++) {
            const int page = __shfl_sync(FULL, iss32, kScorePages * (s & 1) + lane / CPR + 32 * j / CPR);
            constexpr int per = 32 / CPR > 0 ? 32 / CPR : 1;                // rows a step covers
            const int row_j = per * j;
            const uint32_t flip = tile_off<ROWB>(row_j, 0) & 127u, skip = tile_off<ROWB>(row_j, 0) & ~127u;
            // the bounds of a hole are not read
            copy16_or_zero(stage + (lane_dst ^ flip) + skip, lane_src + (uint64_t)(uint32_t)max(page, 0) * page_bytes, page >= 0);
        }
    };
    // ---- query rows, then the first bounds, then the query bytes ----
    uint32_t up[NR][CH][4], down[NR][CH][4];
    Vec16 raw[NR][CH][2];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                raw[r][i][c] = Vec16{{0u, 0u, 0u, 0u}};
                if (g + 8 * r < p.group)
                    raw[r][i][c] = ldg16(reinterpret_cast<const T*>(p.q) + (((int64_t)b * p.num_kv_heads + h) * p.group + g + 8 * r) * D + 16 * (t + 4 * i) + 8 * c);
            }
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) {
        if (s < n_stages) issue(s);
        copies_commit();
    }
    int f_col[NR][2];                                                       // exponents of heads 2t and 2t + 1 (+ 8 r)
    bool wide = false;                                                      // some head's exponent is far from fp32's middle
#pragma unroll
    for (int r = 0; r < NR; r++) {
        float x[CH][16];
        float top = 0.f;                                                    // NaN counts as nothing, here and below
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float2 y = Elem<T>::unpack2(raw[r][i][j >> 2].w[j & 3]);
                x[i][2 * j] = y.x;
                x[i][2 * j + 1] = y.y;
                top = fmax3(top, fabsf(y.x), fabsf(y.y));
            }
        uint32_t amax = __float_as_uint(top);
        amax = max(amax, __shfl_xor_sync(FULL, amax, 1));
        amax = max(amax, __shfl_xor_sync(FULL, amax, 2));
        const int f = bound_exponent(amax);
        const float inv = exp2_int(-f);
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                // adding 1.5 * 2^23 rounds to the nearest even whole number and leaves it in the low byte; NaN becomes 0,
                // infinity 127
                constexpr float magic = 12582912.f;
                uint32_t ub[4], db[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float y = x[i][4 * k + j] * inv;
                    ub[j] = __float_as_uint(fminf(fmaxf(y, 0.f), 127.f) + magic);
                    db[j] = __float_as_uint(fmaxf(fminf(y, 0.f), -127.f) + magic);
                }
                const uint32_t u = __byte_perm(__byte_perm(ub[0], ub[1], 0x0040), __byte_perm(ub[2], ub[3], 0x0040), 0x5410);
                const uint32_t d = __byte_perm(__byte_perm(db[0], db[1], 0x0040), __byte_perm(db[2], db[3], 0x0040), 0x5410);
                up[r][i][k] = u;
                down[r][i][k] = d;
            }
        f_col[r][0] = __shfl_sync(FULL, f, 8 * t);                          // lane 4 (2t) holds head 2t's
        f_col[r][1] = __shfl_sync(FULL, f, 8 * t + 4);
        wide |= f > 60 || (f < -60 && amax != 0);
    }
    wide = __any_sync(FULL, wide);
    float scale[NR][2];                                                     // heads that are not there: -infinity by hand below
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int c = 0; c < 2; c++) scale[r][c] = exp2_int(max(-126, f_col[r][c]));
    uint32_t* keys = p.keys + ((int64_t)b * p.num_kv_heads + h) * p.key_stride;
    uint32_t key = kKeyHole;                                                // of this lane's page of the window
    for (int s = 0; s < n_stages; s++) {
        if (s + STAGES - 1 < n_stages) issue(s + STAGES - 1);
        copies_commit();
        copies_wait<STAGES - 1>();
        __syncwarp();
        const uint32_t stage = ring + (s % STAGES) * STAGE;
        int acc[NR][4] = {};
#pragma unroll
        for (int i = 0; i < 2 * CH; i++) {                                  // upper bounds, then lower
            const uint4 a = lds128(stage + tile_off<ROWB>(g, t + 4 * i)), c = lds128(stage + tile_off<ROWB>(g + 8, t + 4 * i));
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const uint32_t* q = i < CH ? up[r][i % CH] : down[r][i % CH];
                mma_s8(acc[r], a.x, c.x, a.y, c.y, q[0], q[1]);
                mma_s8(acc[r], a.z, c.z, a.w, c.w, q[2], q[3]);
            }
        }
        __syncwarp();                                                       // the stage is free for the next request
        // pages g and g + 8 of the stage, heads 2t and 2t + 1 (+ 8 r)
        float mine = 0.f;                                                   // of this lane's page, if it is in this stage
        const int from = 4 * (lane & 7);                                    // a lane of that page's row of the tile
        if (!wide) {
            // whole number * 2^f is exact in fp32 here, and the maximum over the heads may come before 2^e
            float best[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float x = -INFINITY;
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int c = 0; c < 2; c++)
                        if (2 * t + c + 8 * r < p.group) x = fmaxf(x, (float)acc[r][2 * k + c] * scale[r][c]);
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 1));
                best[k] = fmaxf(x, __shfl_xor_sync(FULL, x, 2));
            }
            const float b0 = __shfl_sync(FULL, best[0], from), b1 = __shfl_sync(FULL, best[1], from);
            mine = ((lane & 8) ? b1 : b0) * exp2_int(e32);
        } else {                                                            // the same in fp64, whose range holds every case
            double best[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                double x = -INFINITY;
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int c = 0; c < 2; c++)
                        if (2 * t + c + 8 * r < p.group) x = fmax(x, ldexp((double)acc[r][2 * k + c], f_col[r][c]));
                x = fmax(x, __shfl_xor_sync(FULL, x, 1));
                best[k] = fmax(x, __shfl_xor_sync(FULL, x, 2));
            }
            const double b0 = __shfl_sync(FULL, best[0], from), b1 = __shfl_sync(FULL, best[1], from);
            mine = (float)ldexp((lane & 8) ? b1 : b0, e32);
        }
        if (lane >> 4 == (s & 1)) key = ordered(mine);
        if ((s & 1) || s == n_stages - 1) {                                 // a window of 32 pages is done
            const int idx = begin + (s & ~1) * kScorePages + lane;
            if (idx < last)
                keys[idx] = page32 < 0 ? kKeyHole : (idx < p.first_pages || idx >= n - p.last_pages) ? kKeyForced : key;
            page32 = next32;
            e32 = next_e;
            next32 = checked(page_ids(begin + (s & ~1) * kScorePages + 64));
            next_e = exponent_of(next32);
        }
    }
}

// One CTA per (KV head, sequence): the top_pages largest keys (ties: lowest page), pages ascending, -1 behind them.
// The k-th largest key is found by 8-bit digits from the first bit in which the keys differ (scores of one query share
// their exponent: counting digits from the top would put them all into one bin), each pass over the keys that share the
// digits found so far; as soon as a bin's keys are all needed or none is, the rest of the digits does not matter.
// Then every thread takes a run of pages and one scan gives each its places.
constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32;
__global__ void __launch_bounds__(kSelectThreads) page_select_kernel(const SelectParams p, int smem_keys) {
    extern __shared__ uint32_t s_keys[];
    __shared__ int s_bins[256];
    __shared__ int s_int[2][kSelectWarps];
    __shared__ uint32_t s_min[kSelectWarps], s_max[kSelectWarps];
    __shared__ int s_pick[2];                                               // digit of the cut, keys still needed in its bin
    pdl_wait();
    pdl_launch_dependents();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int64_t pair = (int64_t)b * p.num_kv_heads + h;
    const int row = __ldg(p.rows + b);
    const int len = min(__ldg(p.kv_len + b), p.max_kv_len);
    const int n = len <= 0 || row < 0 || row >= p.max_rows ? 0 : min((len - 1) / p.page_size + 1, p.table_stride);
    const uint32_t* keys = p.keys + pair * p.key_stride;
    int32_t* sel = p.sel + pair * p.top_pages;
    // ---- keys into shared memory; how many are resident, how many forced, and the others' range ----
    int resident = 0, forced = 0;
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll 4
    for (int i = tid; i < n; i += kSelectThreads) {
        const uint32_t k = __ldcg(keys + i);
        if (i < smem_keys) s_keys[i] = k;
        resident += k != kKeyHole;
        forced += k == kKeyForced;
        if (k != kKeyHole && k != kKeyForced) {
            lo = min(lo, k);
            hi = max(hi, k);
        }
    }
    resident = __reduce_add_sync(FULL, resident);
    forced = __reduce_add_sync(FULL, forced);
    lo = __reduce_min_sync(FULL, lo);
    hi = __reduce_max_sync(FULL, hi);
    if (lane == 0) {
        s_int[0][w] = resident;
        s_int[1][w] = forced;
        s_min[w] = lo;
        s_max[w] = hi;
    }
    for (int i = tid; i < 256; i += kSelectThreads) s_bins[i] = 0;
    __syncthreads();
    resident = forced = 0;
#pragma unroll
    for (int i = 0; i < kSelectWarps; i++) {
        resident += s_int[0][i];
        forced += s_int[1][i];
        lo = min(lo, s_min[i]);
        hi = max(hi, s_max[i]);
    }
    auto key_at = [&](int i) { return i < smem_keys ? s_keys[i] : __ldcg(keys + i); };
    const int k = min(p.top_pages, resident);
    // Taken are keys > cut_hi, and of those in [cut_lo, cut_hi] the first `ties` by page (more than there are: all).
    uint32_t cut_lo = 1, cut_hi = 0;                                        // everything resident
    int ties = 0;
    if (resident > k) {
        int need = k - forced;                                              // of the keys in [lo, hi]
        if (need <= 0 || lo > hi) {
            cut_lo = cut_hi = kKeyForced;                                   // forced ones only, the first k
            ties = k;
        } else {
            int shift = lo == hi ? 0 : 32 - __clz(lo ^ hi);                 // bits from here on down differ
            uint32_t prefix = shift >= 32 ? 0u : hi >> shift << shift;      // shared by all candidates
            cut_lo = prefix;
            cut_hi = hi;
            while (shift > 0) {
                const int down = shift < 8 ? 0 : shift - 8, bits = shift - down;
                for (int i = tid; i < n; i += kSelectThreads) {
                    const uint32_t key = key_at(i);
                    if (key >= cut_lo && key <= cut_hi) atomicAdd(&s_bins[(key >> down) & ((1u << bits) - 1)], 1);
                }
                __syncthreads();
                if (w == 0) {                                               // lane's bins: 255 - 8 lane .. 248 - 8 lane, from the top
                    int c[8], sum = 0;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        c[i] = s_bins[255 - 8 * lane - i];
                        sum += c[i];
                    }
                    int above = sum;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int v = __shfl_up_sync(FULL, above, o);
                        if (lane >= o) above += v;
                    }
                    above -= sum;                                           // keys in bins above the lane's
                    if (above < need && above + sum >= need) {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            if (above < need && above + c[i] >= need) {
                                s_pick[0] = 255 - 8 * lane - i;
                                s_pick[1] = need - above;
                            }
                            above += c[i];
                        }
                    }
                }
                __syncthreads();
                const int digit = s_pick[0], in_bin = s_bins[digit];
                need = s_pick[1];
                __syncthreads();
                for (int i = tid; i < 256; i += kSelectThreads) s_bins[i] = 0;
                __syncthreads();
                cut_lo |= (uint32_t)digit << down;
                cut_hi = cut_lo | ((1u << down) - 1);
                shift = down;
                if (need == in_bin) break;                                  // the whole bin is taken
            }
            ties = need;
        }
    }
    // ---- places: a run of pages per thread ----
    const int run = (n + kSelectThreads - 1) / kSelectThreads, i0 = min(n, tid * run), i1 = min(n, i0 + run);
    const bool all = resident == k;
    int gt = 0, eq = 0;
    for (int i = i0; i < i1; i++) {
        const uint32_t key = key_at(i);
        gt += all ? key != kKeyHole : key > cut_hi;
        eq += !all && key >= cut_lo && key <= cut_hi;
    }
    int gt_in = gt, eq_in = eq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(FULL, gt_in, o), c = __shfl_up_sync(FULL, eq_in, o);
        if (lane >= o) {
            gt_in += a;
            eq_in += c;
        }
    }
    __syncthreads();
    if (lane == 31) {
        s_int[0][w] = gt_in;
        s_int[1][w] = eq_in;
    }
    __syncthreads();
    int gt_at = gt_in - gt, eq_at = eq_in - eq;
    for (int i = 0; i < w; i++) {
        gt_at += s_int[0][i];
        eq_at += s_int[1][i];
    }
    for (int i = i0; i < i1; i++) {
        const uint32_t key = key_at(i);
        const bool is_gt = all ? key != kKeyHole : key > cut_hi, is_eq = !all && key >= cut_lo && key <= cut_hi;
        if (is_gt || (is_eq && eq_at < ties)) sel[gt_at + min(eq_at, ties)] = i;
        gt_at += is_gt;
        eq_at += is_eq;
    }
    for (int i = k + tid; i < p.top_pages; i += kSelectThreads) sel[i] = -1;
}

template <bool POOL8, typename T>
cudaError_t launch_bounds_d(const BoundsParams& p, bool split, int head_dim, dim3 grid, cudaStream_t s) {
    switch (head_dim) {
        case 64: return split ? launch_pdl(bounds_kernel<POOL8, T, 64, true>, grid, dim3(256), 0, s, p)
                              : launch_pdl(bounds_kernel<POOL8, T, 64, false>, grid, dim3(256), 0, s, p);
        case 128: return split ? launch_pdl(bounds_kernel<POOL8, T, 128, true>, grid, dim3(256), 0, s, p)
                              : launch_pdl(bounds_kernel<POOL8, T, 128, false>, grid, dim3(256), 0, s, p);
        case 256: return split ? launch_pdl(bounds_kernel<POOL8, T, 256, true>, grid, dim3(256), 0, s, p)
                              : launch_pdl(bounds_kernel<POOL8, T, 256, false>, grid, dim3(256), 0, s, p);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T, int D>
cudaError_t launch_score(const SelectParams& p, int num_sms, cudaStream_t s) {
    const int pages = min((p.max_kv_len - 1) / p.page_size + 1, p.table_stride);
    int heads = kScoreWarps;
    while (p.num_kv_heads % heads) heads >>= 1;
    // 32 pages a warp; more (the query bytes are made once a warp) while CTAs for three turns of three an SM remain
    int per_cta = 32 * (kScoreWarps / heads);
    const int64_t ctas = (int64_t)(p.num_kv_heads / heads) * p.n_seq;
    while (per_cta < 4096 && (pages + 2 * per_cta - 1) / (2 * per_cta) * ctas >= 9 * num_sms) per_cta *= 2;
    const dim3 grid((pages + per_cta - 1) / per_cta, p.num_kv_heads / heads, p.n_seq);
    constexpr size_t smem = (size_t)kScoreWarps * kScoreStages<D> * kScorePages * 2 * D;
    auto kernel = p.group > 8 ? page_score_kernel<T, D, true> : page_score_kernel<T, D, false>;
    static std::atomic<bool> configured[64][2];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !configured[dev][p.group > 8].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev][p.group > 8].store(true, std::memory_order_release);
    }
    return launch_pdl(kernel, grid, dim3(kScoreWarps * 32), smem, s, p, per_cta, heads);
}

}  // namespace

cudaError_t launch_bounds(const BoundsParams& p, bool pool8, int head_dim, int dtype, int num_layers, int num_sms, cudaStream_t stream) {
    if (p.n_items <= 0 || num_layers <= 0) return cudaSuccess;
    const int64_t items = (int64_t)p.n_items * p.num_kv_heads;
    const bool split = p.rows == nullptr && items * num_layers < 64 * num_sms;   // 64 warps an SM
    const int64_t blocks = split ? items : (items + 7) / 8;
    if (blocks > 0x7fffffff || num_layers > 65535) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)blocks, num_layers);
    if (pool8) return launch_bounds_d<true, __half>(p, split, head_dim, grid, stream);
    return dtype == DRKV_DTYPE_F16 ? launch_bounds_d<false, __half>(p, split, head_dim, grid, stream)
                                   : launch_bounds_d<false, __nv_bfloat16>(p, split, head_dim, grid, stream);
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
    // keys beyond 11 776 (46 KB) of a sequence are read from global memory (L2) in every round
    const int pages = p.max_kv_len > 0 ? min((p.max_kv_len - 1) / p.page_size + 1, p.table_stride) : 0;
    const int smem_keys = pages < 11776 ? pages : 11776;
    return launch_pdl(page_select_kernel, dim3(p.num_kv_heads, p.n_seq), dim3(kSelectThreads), (size_t)smem_keys * 4, stream, p, smem_keys);
}

}  // namespace drkv
