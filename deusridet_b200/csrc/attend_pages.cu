// attend_pages.cu — decode attention over the 8-bit pool, and over a list of pages per KV head (either pool).
//
//   o_h = sum_j softmax_j(scale q_h . k_j) v_j       over the keys of the sequence, or of the listed pages only
// The bytes are the cost: (D + 1) per K or V row of the 8-bit pool, 2 D of the 16-bit one, each read once per KV head; the
// 4 D flops per key and query head ride on mma.sync tiles far from their limit (a GQA group fills one 8-column tile).
//
// Split: the keys of all (sequence, KV head) pairs form one line of 16-key groups.  Every warp of a persistent grid takes
// an equal stretch of it (at least kMinShare groups), whatever the lengths are: ragged batches need no queue and no
// tail.  A pair that lies inside one stretch is finished by its warp; one that is cut leaves a partial (m, l, o) per
// stretch, at most two a warp, and a second small kernel merges them in a fixed order (results do not depend on timing).
// Warps of one CTA take stretches far apart, so that a short line still spreads over all SMs.
//
// A warp brings its groups into a private ring of shared memory by cp.async (16 bytes a lane, L1 bypassed), kStages - 1
// groups ahead, and reads them as matrix operands without ldmatrix: contraction order is free, so a lane takes whole
// 16-byte chunks of a row.  Tokens are the M dimension, S^T = K Q^T (A = K rows, B = the group's queries, 8 columns) and
// O^T = V^T P^T (A = V^T, two keys' bytes interleaved by prmt): half the tiles of the usual orientation, where 16 query
// rows would be half empty.  P turns from the accumulator layout into the operand layout by movmatrix.  e4m3 operands
// become f16 two at a time (cvt.rn.f16x2.e4m3x2, exact).
//
// Scales of the 8-bit rows stay exponents.  K's multiply the score.  V's multiply the weight: with E the largest exponent
// seen so far, weights are p * 2^(ev - E + 15) <= 2^15 in f16, full precision down to 2^-29 of the largest; o carries 2^E.
// bf16 queries are scaled by a power of two per head into f16 (8 significant bits fit; exact unless an element is below
// 2^-27 of its row's maximum).  Scores, maxima, sums and outputs accumulate in fp32.
// P in the PV product: f16 hi + lo terms (22 bits) where the output is f16, bf16 hi + lo (16 bits) for a bf16 pool,
// one f16 term (2^-11) where the pool is 8-bit and the output bf16 (2^-8 steps).
#include <atomic>

#include "kernels.hpp"
#include "kv_common.cuh"
#include "sm100_primitives.cuh"

namespace drkv {

namespace {

constexpr int kMinShare = 4;          // 16-key groups: shorter stretches cost more in partials than they save
constexpr float kNoKey = -1.0e30f;    // running maximum before any key

// Warps per CTA (one CTA per SM) and groups in a warp's ring.
template <bool POOL8, int D> struct Ring;
template <> struct Ring<true, 64>   { static constexpr int kWarps = 16, kStages = 4; };   // 132 KB
template <> struct Ring<true, 128>  { static constexpr int kWarps = 16, kStages = 3; };   // 198 KB
template <> struct Ring<true, 256>  { static constexpr int kWarps = 8, kStages = 3; };    // 197 KB
template <> struct Ring<false, 64>  { static constexpr int kWarps = 16, kStages = 3; };   // 192 KB
template <> struct Ring<false, 128> { static constexpr int kWarps = 8, kStages = 3; };    // 192 KB
template <> struct Ring<false, 256> { static constexpr int kWarps = 6, kStages = 2; };    // 192 KB

// A tile is 16 rows of ROWB bytes in shared memory; chunks of 16 bytes are permuted so that both access patterns are free
// of bank conflicts: rows (g) x chunks (t) for K, rows (2t) x chunks (g) for V, g = lane / 4, t = lane % 4.
template <int ROWB>
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
    if (ROWB == 64)                    // two rows share a 128-byte line
        return (row >> 1) * 128 + (((((row & 1) << 2) | chunk) ^ (((row >> 1) & 3) << 1)) << 4);
    return row * ROWB + ((chunk ^ ((((row >> 1) & 3) << 1) ^ ((row & 1) << 2))) << 4);
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
// 16 bytes from global to shared memory, zeros where !live
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The work split, left by the first kernel for the second: share, then the line's prefix sums over the sequences.
struct Split {
    int share;
    int cum[kMaxDecodeSeqs + 1];
};
constexpr size_t kSplitFloats = (sizeof(Split) + 255) / 256 * 64;

struct PartialView {                   // slot = 2 * warp + (the stretch's first piece ? 0 : 1), row = head of the group
    float *o, *m, *l;
    __host__ __device__ PartialView(float* scratch, size_t slots, int group, int d) {
        o = scratch + kSplitFloats;
        m = o + slots * group * d;
        l = m + slots * group;
    }
};

// Groups of a pair of sequence b.  A list has at most as many entries as the sequence has pages.
__device__ __forceinline__ int pair_groups(const AttendPagesParams& p, int b, bool list) {
    int len = __ldg(p.kv_len + b);
    len = min(len, p.max_kv_len);
    const int row = __ldg(p.rows + b);
    if (len <= 0 || row < 0 || row >= p.max_rows) return 0;
    if (!list) return (len + 15) >> 4;
    const int pages = (len - 1) / p.page_size + 1;
    return min(pages, p.list_len) * (p.page_size >> 4);
}

template <bool POOL8, typename T, int D, int NQ, bool LIST>
__global__ void __launch_bounds__(Ring<POOL8, D>::kWarps * 32, 1) attend_pages_kernel(const AttendPagesParams p) {
    constexpr int WARPS = Ring<POOL8, D>::kWarps, STAGES = Ring<POOL8, D>::kStages, THREADS = WARPS * 32;
    using TM = typename std::conditional<POOL8, __half, T>::type;           // matrix operand type
    constexpr bool F16 = std::is_same<TM, __half>::value;
    constexpr bool LO = !(POOL8 && std::is_same<T, __nv_bfloat16>::value);
    constexpr int ROWB = D * (POOL8 ? 1 : 2), CPR = ROWB / 16, TILE = 16 * ROWB;
    constexpr int SLOT = 2 * TILE + (POOL8 ? 32 : 0);
    constexpr int KSTEPS = D / 16, MT = D / 16;
    constexpr int KCH = CPR / 4;                                            // K chunks a lane reads of a row
    constexpr int EPL = POOL8 ? (D == 64 ? 8 : 16) : 8;                     // V elements a lane reads of a row at once
    constexpr int VCH = D / (8 * EPL);
    constexpr int WS = F16 ? 15 : 0;                                        // weights carry 2^WS
    constexpr uint32_t FULL = 0xffffffffu;

    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_warp_tot[WARPS];
    __shared__ int2 s_meta[WARPS][STAGES];                                  // pair, visible keys of the group
    int* cum = reinterpret_cast<int*>(smem + WARPS * STAGES * SLOT);        // [n_seq + 1]

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch_dependents();

    // ---- prefix sums of the line over the sequences ----
    {
        const int per = (p.n_seq + THREADS - 1) / THREADS;
        const int lo = min(tid * per, p.n_seq), hi = min(lo + per, p.n_seq);
        int local = 0;
        for (int b = lo; b < hi; b++) local += pair_groups(p, b, LIST) * p.num_kv_heads;
        int incl = local;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(FULL, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) s_warp_tot[w] = incl;
        __syncthreads();
        int run = incl - local;
        for (int i = 0; i < w; i++) run += s_warp_tot[i];
        for (int b = lo; b < hi; b++) {
            cum[b] = run;
            run += pair_groups(p, b, LIST) * p.num_kv_heads;
        }
        if (tid == THREADS - 1) cum[p.n_seq] = run;
        __syncthreads();
    }
    const int total = cum[p.n_seq];
    const int n_warps = (int)gridDim.x * WARPS;
    const int share = max(kMinShare, (total + n_warps - 1) / n_warps);
    if (blockIdx.x == 0) {
        Split* split = reinterpret_cast<Split*>(p.scratch);
        if (tid == 0) split->share = share;
        for (int b = tid; b <= p.n_seq; b += THREADS) split->cum[b] = cum[b];
    }
    const int gw = w * (int)gridDim.x + (int)blockIdx.x;
    const int64_t lo64 = (int64_t)gw * share;
    if (lo64 >= total) return;                                              // no block-wide barrier below
    const int lo = (int)lo64, n = min(share, total - lo);

    // ---- where a group of the line lies: lane i describes group (window's first) + i ----
    struct Where { int pair, tok, valid, page; };
    auto locate = [&](int idx) -> Where {
        Where r{-1, 0, 0, -1};
        if (idx >= n) return r;
        const int f = lo + idx;
        int b = 0, e = p.n_seq;                                             // largest b with cum[b] <= f
        while (e - b > 1) {
            const int mid = (b + e) >> 1;
            if (cum[mid] <= f) b = mid; else e = mid;
        }
        const int groups = (cum[b + 1] - cum[b]) / p.num_kv_heads;
        const int rem = f - cum[b], h = rem / groups, i = rem - h * groups;
        r.pair = b * p.num_kv_heads + h;
        const int len = min(__ldg(p.kv_len + b), p.max_kv_len);
        const int per_page = p.page_size >> 4;
        int logical = i / per_page;
        const int sub = i - logical * per_page;
        if (LIST) logical = __ldg(p.list + (int64_t)r.pair * p.list_len + logical);
        if (logical < 0 || logical >= p.table_stride) return r;
        const int64_t tok = (int64_t)logical * p.page_size + sub * 16;
        if (tok >= len) return r;
        r.tok = (int)tok;
        r.page = __ldg(p.tables + (int64_t)__ldg(p.rows + b) * p.table_stride + logical);
        if (r.page >= p.max_pages) {
            atomicExch(p.error_word, (int)KERR_BAD_PAGE);
            r.page = -1;
        }
        if (r.page >= 0) r.valid = min(16, len - r.tok);
        return r;
    };
    Where cur = locate(lane), next = cur;
    const uint32_t ring = smem_u32(smem) + w * STAGES * SLOT;

    auto issue = [&](int idx) {                                             // requests group idx of the stretch
        const int wl = idx & 31;
        if (wl == 0) {
            if (idx > 0) cur = next;
            if (idx + 32 < n) next = locate(idx + 32 + lane);               // used 32 groups from now
        }
        const int pair = __shfl_sync(FULL, cur.pair, wl), tok = __shfl_sync(FULL, cur.tok, wl);
        const int valid = __shfl_sync(FULL, cur.valid, wl), page = __shfl_sync(FULL, cur.page, wl);
        const int stage = idx % STAGES;
        if (lane == 0) s_meta[w][stage] = make_int2(pair, valid);
        if (valid > 0) {
            const uint32_t dst = ring + stage * SLOT;
            const int h = pair % p.num_kv_heads;
            const int64_t row0 = (int64_t)h * p.page_size + tok % p.page_size;
            const uint8_t* block = p.pool + (int64_t)page * p.block_bytes;
            const uint8_t* k = block + row0 * ROWB;
            const uint8_t* v = k + p.plane_bytes;
#pragma unroll
            for (int c = lane; c < 16 * CPR; c += 32) {
                const int row = c / CPR;
                const uint32_t off = tile_off<ROWB>(row, c % CPR);
                copy16(dst + off, k + 16 * c, row < valid);
                copy16(dst + TILE + off, v + 16 * c, row < valid);          // hidden rows are zeros: they meet zero weights
            }
            if (POOL8 && lane < 2) copy16(dst + 2 * TILE + 16 * lane, block + 2 * p.plane_bytes + lane * p.exp_plane_bytes + row0, true);
        }
    };

    // ---- state of the pair being attended ----
    uint32_t qf[NQ][KSTEPS][2];
    float qs[NQ][2];                                                        // score factor of heads 2t and 2t + 1
    float o[NQ][MT][4], m[NQ][2], l[NQ][2];
    int big_e = -127, cur_pair = -1, seg_begin = 0;

    auto begin_pair = [&](int pair, int f) {
        cur_pair = pair;
        seg_begin = f;
        const int b = pair / p.num_kv_heads, h = pair - b * p.num_kv_heads;
        const T* q = reinterpret_cast<const T*>(p.q) + ((int64_t)b * p.num_kv_heads + h) * p.group * D;
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            const int head = nq * 8 + g;
            const bool live = head < p.group;
            const T* qh = q + (int64_t)head * D;
            float own_scale = p.scale_log2;
            if (POOL8) {
                // lane t owns dims 16 (t + 4 i) .. + 15, word w of a chunk is K step 4 i + w
                uint32_t raw[KCH][8];
                uint32_t amax = 0;
#pragma unroll
                for (int i = 0; i < KCH; i++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        Vec16 v = Vec16{{0u, 0u, 0u, 0u}};
                        if (live) v = ldg16(qh + 16 * (t + 4 * i) + 8 * c);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            raw[i][4 * c + j] = v.w[j];
                            const float2 f2 = Elem<T>::unpack2(v.w[j]);
                            amax = max(amax, max(__float_as_uint(f2.x) & 0x7fffffffu, __float_as_uint(f2.y) & 0x7fffffffu));
                        }
                    }
                float to16 = 1.f;
                if (!std::is_same<T, __half>::value) {                      // maximum into [2^13, 2^14)
                    amax = max(amax, __shfl_xor_sync(FULL, amax, 1));
                    amax = max(amax, __shfl_xor_sync(FULL, amax, 2));
                    const int e = max(-100, min(126, (int)(amax >> 23) - 127));
                    to16 = exp2_int(13 - e);
                    own_scale *= exp2_int(e - 13);
                }
#pragma unroll
                for (int i = 0; i < KCH; i++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float2 f2 = Elem<T>::unpack2(raw[i][j]);
                        qf[nq][(4 * i + (j >> 1)) % KSTEPS][j & 1] = Elem<__half>::pack2(f2.x * to16, f2.y * to16);
                    }
            } else {
                // lane t owns dims 8 (t + 4 i) .. + 7: K steps 2 i and 2 i + 1
#pragma unroll
                for (int i = 0; i < KCH; i++) {
                    Vec16 v = Vec16{{0u, 0u, 0u, 0u}};
                    if (live) v = ldg16(qh + 8 * (t + 4 * i));
#pragma unroll
                    for (int j = 0; j < 4; j++) qf[nq][(2 * i + (j >> 1)) % KSTEPS][j & 1] = v.w[j];
                }
            }
            qs[nq][0] = __shfl_sync(FULL, own_scale, 8 * t);                // lane 4 (2t) holds head 2t's
            qs[nq][1] = __shfl_sync(FULL, own_scale, 8 * t + 4);
            m[nq][0] = m[nq][1] = kNoKey;
            l[nq][0] = l[nq][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) o[nq][mt][0] = o[nq][mt][1] = o[nq][mt][2] = o[nq][mt][3] = 0.f;
        }
        big_e = -127;
    };

    auto end_pair = [&](int f_end) {
        const int b = cur_pair / p.num_kv_heads, h = cur_pair - b * p.num_kv_heads;
        const int groups = (cum[b + 1] - cum[b]) / p.num_kv_heads;
        const int start = cum[b] + h * groups;
        const bool whole = seg_begin == start && f_end == start + groups;
        const PartialView parts(p.scratch, 2 * (size_t)n_warps, p.group, D);
        const int64_t slot = 2 * (int64_t)gw + (seg_begin == lo ? 0 : 1);
        const float unit = POOL8 ? exp2_int(big_e) : 1.f;
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float sum = l[nq][c];
                sum += __shfl_xor_sync(FULL, sum, 4);
                sum += __shfl_xor_sync(FULL, sum, 8);
                sum += __shfl_xor_sync(FULL, sum, 16);
                const int head = nq * 8 + 2 * t + c;
                if (head >= p.group) continue;
                const float f = (whole ? 1.f / sum : 1.f) * (F16 ? 0x1p-15f : 1.f);
                const int64_t row = slot * p.group + head;
                if (!whole && g == 0) {
                    parts.m[row] = m[nq][c];
                    parts.l[row] = sum;
                }
#pragma unroll
                for (int j = 0; j < VCH; j++) {
                    const int dim = (g + 8 * j) * EPL;
                    float x[EPL];
#pragma unroll
                    for (int i = 0; i < EPL / 2; i++) {
                        x[2 * i] = o[nq][j * (EPL / 2) + i][c] * f * unit;
                        x[2 * i + 1] = o[nq][j * (EPL / 2) + i][2 + c] * f * unit;
                    }
                    if (whole) {
                        if (!(sum != 0.f)) continue;                        // no visible key: the row stays as it is
                        T* dst = reinterpret_cast<T*>(p.out) + (((int64_t)b * p.num_kv_heads + h) * p.group + head) * D + dim;
#pragma unroll
                        for (int i = 0; i < EPL; i += 8) {
                            Vec16 v;
#pragma unroll
                            for (int k = 0; k < 4; k++) v.w[k] = Elem<T>::pack2(x[i + 2 * k], x[i + 2 * k + 1]);
                            stg16(dst + i, v);
                        }
                    } else {
                        float* dst = parts.o + row * D + dim;
#pragma unroll
                        for (int i = 0; i < EPL; i += 4)
                            *reinterpret_cast<float4*>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                    }
                }
            }
    };

    auto attend_group = [&](uint32_t tile, int valid) {
        // ---- scores: tokens g and g + 8, heads 2t and 2t + 1 of every 8-head tile ----
        float s[NQ][4];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) s[nq][0] = s[nq][1] = s[nq][2] = s[nq][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KCH; i++) {
            const uint4 ka = lds128(tile + tile_off<ROWB>(g, t + 4 * i)), kb = lds128(tile + tile_off<ROWB>(g + 8, t + 4 * i));
            const uint32_t a[4] = {ka.x, ka.y, ka.z, ka.w}, b[4] = {kb.x, kb.y, kb.z, kb.w};
            if (POOL8) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t a0 = e4m3x2_to_f16x2(a[j] & 0xffffu), a2 = e4m3x2_to_f16x2(a[j] >> 16);
                    const uint32_t a1 = e4m3x2_to_f16x2(b[j] & 0xffffu), a3 = e4m3x2_to_f16x2(b[j] >> 16);
#pragma unroll
                    for (int nq = 0; nq < NQ; nq++)
                        mma16816<TM>(s[nq], a0, a1, a2, a3, qf[nq][(4 * i + j) % KSTEPS][0], qf[nq][(4 * i + j) % KSTEPS][1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int nq = 0; nq < NQ; nq++)
                        mma16816<TM>(s[nq], a[2 * j], b[2 * j], a[2 * j + 1], b[2 * j + 1], qf[nq][(2 * i + j) % KSTEPS][0],
                                     qf[nq][(2 * i + j) % KSTEPS][1]);
            }
        }
        const bool see0 = g < valid, see1 = g + 8 < valid;
        float ks0 = 1.f, ks1 = 1.f;
        int ev0 = 0, ev1 = 0, new_e = big_e;
        if (POOL8) {
            ks0 = exp2_int((int)lds8(tile + 2 * TILE + g) - 127);
            ks1 = exp2_int((int)lds8(tile + 2 * TILE + g + 8) - 127);
            ev0 = (int)lds8(tile + 2 * TILE + 16 + g) - 127;
            ev1 = (int)lds8(tile + 2 * TILE + 24 + g) - 127;
            new_e = max(big_e, __reduce_max_sync(FULL, max(see0 ? ev0 : -127, see1 ? ev1 : -127)));
        }
        float mx[NQ][2];
        bool grow = new_e > big_e;
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                s[nq][c] = see0 ? s[nq][c] * (ks0 * qs[nq][c]) : -INFINITY;
                s[nq][2 + c] = see1 ? s[nq][2 + c] * (ks1 * qs[nq][c]) : -INFINITY;
                float x = fmaxf(s[nq][c], s[nq][2 + c]);
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 4));
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 8));
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 16));
                mx[nq][c] = fmaxf(m[nq][c], x);
                grow |= mx[nq][c] > m[nq][c];
            }
        }
        if (__any_sync(FULL, grow)) {
            // 2^(old - new E) in two factors: the difference may be 247
            const int de = big_e - new_e;
            const float e1 = exp2_int(max(de, -126)), e2 = exp2_int(max(de - max(de, -126), -126));
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
                const float f0 = fast_exp2(m[nq][0] - mx[nq][0]), f1 = fast_exp2(m[nq][1] - mx[nq][1]);
                m[nq][0] = mx[nq][0];
                m[nq][1] = mx[nq][1];
                l[nq][0] *= f0;
                l[nq][1] *= f1;
                const float r0 = POOL8 ? f0 * e1 * e2 : f0, r1 = POOL8 ? f1 * e1 * e2 : f1;
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    o[nq][mt][0] *= r0;
                    o[nq][mt][1] *= r1;
                    o[nq][mt][2] *= r0;
                    o[nq][mt][3] *= r1;
                }
            }
            big_e = new_e;
        }
        // ---- weights ----
        float vs0 = F16 ? 0x1p15f : 1.f, vs1 = vs0;
        if (POOL8) {
            vs0 = exp2_int(max(min(ev0, big_e) - big_e + WS, -127));
            vs1 = exp2_int(max(min(ev1, big_e) - big_e + WS, -127));
        }
        uint32_t pf[NQ][2], pl[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            const float p00 = fast_exp2(s[nq][0] - m[nq][0]), p01 = fast_exp2(s[nq][1] - m[nq][1]);
            const float p10 = fast_exp2(s[nq][2] - m[nq][0]), p11 = fast_exp2(s[nq][3] - m[nq][1]);
            l[nq][0] += p00 + p10;
            l[nq][1] += p01 + p11;
            const uint32_t h0 = Elem<TM>::pack2(p00 * vs0, p01 * vs0), h1 = Elem<TM>::pack2(p10 * vs1, p11 * vs1);
            pf[nq][0] = transpose8x8(h0);
            pf[nq][1] = transpose8x8(h1);
            if (LO) {
                const float2 a = Elem<TM>::unpack2(h0), b = Elem<TM>::unpack2(h1);
                pl[nq][0] = transpose8x8(Elem<TM>::pack2(p00 * vs0 - a.x, p01 * vs0 - a.y));
                pl[nq][1] = transpose8x8(Elem<TM>::pack2(p10 * vs1 - b.x, p11 * vs1 - b.y));
            }
        }
        // ---- O^T += V^T P^T: keys 2t, 2t + 1, 2t + 8, 2t + 9; dims (g + 8 j) EPL + 0 .. EPL - 1 ----
        const uint32_t vt = tile + TILE;
        auto pv = [&](int mt, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
                mma16816<TM>(o[nq][mt], a0, a1, a2, a3, pf[nq][0], pf[nq][1]);
                if (LO) mma16816<TM>(o[nq][mt], a0, a1, a2, a3, pl[nq][0], pl[nq][1]);
            }
        };
#pragma unroll
        for (int j = 0; j < VCH; j++) {
            constexpr int WORDS = EPL * (POOL8 ? 1 : 2) / 4;
            uint32_t v[4][WORDS];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 2 * t + (r & 1) + 8 * (r >> 1);
                if constexpr (WORDS == 4) {
                    const uint4 x = lds128(vt + tile_off<ROWB>(row, g + 8 * j));
                    v[r][0] = x.x;
                    v[r][1] = x.y;
                    v[r][2] = x.z;
                    v[r][3] = x.w;
                } else {                                                    // 64-byte rows: 8 bytes a lane
                    const uint2 x = lds64(vt + tile_off<ROWB>(row, g >> 1) + 8 * (g & 1));
                    v[r][0] = x.x;
                    v[r][1] = x.y;
                }
            }
#pragma unroll
            for (int i = 0; i < WORDS; i++) {
                if (POOL8) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const uint32_t x = __byte_perm(v[0][i], v[1][i], half ? 0x7362 : 0x5140);
                        const uint32_t y = __byte_perm(v[2][i], v[3][i], half ? 0x7362 : 0x5140);
                        pv(j * (EPL / 2) + 2 * i + half, e4m3x2_to_f16x2(x & 0xffffu), e4m3x2_to_f16x2(x >> 16),
                           e4m3x2_to_f16x2(y & 0xffffu), e4m3x2_to_f16x2(y >> 16));
                    }
                } else {
                    pv(j * (EPL / 2) + i, __byte_perm(v[0][i], v[1][i], 0x5410), __byte_perm(v[0][i], v[1][i], 0x7632),
                       __byte_perm(v[2][i], v[3][i], 0x5410), __byte_perm(v[2][i], v[3][i], 0x7632));
                }
            }
        }
    };

    // ---- the stretch ----
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) {
        if (i < n) issue(i);
        copies_commit();
    }
    for (int i = 0; i < n; i++) {
        if (i + STAGES - 1 < n) issue(i + STAGES - 1);
        copies_commit();
        copies_wait<STAGES - 1>();
        __syncwarp();
        const int2 meta = s_meta[w][i % STAGES];
        if (meta.x != cur_pair) {
            if (cur_pair >= 0) end_pair(lo + i);
            begin_pair(meta.x, lo + i);
        }
        if (meta.y > 0) attend_group(ring + (i % STAGES) * SLOT, meta.y);
        __syncwarp();                                                       // the slot is free for the next request
    }
    end_pair(lo + n);
}

// One CTA per (query head, sequence): merges what the stretches left of a pair that was cut.
template <typename T, int D>
__global__ void __launch_bounds__(512) merge_pieces_kernel(const AttendPagesParams p, int n_warps) {
    constexpr int LPR = D / 4;                                              // lanes per partial row
    __shared__ float s_red[16];
    __shared__ float4 s_o[512];
    __shared__ float s_l[512 / LPR];
    pdl_wait();
    pdl_launch_dependents();
    const Split* split = reinterpret_cast<const Split*>(p.scratch);
    const int b = blockIdx.y, hq = blockIdx.x, h = hq / p.group, head = hq - h * p.group;
    const int share = split->share, c0 = split->cum[b];
    const int groups = (split->cum[b + 1] - c0) / p.num_kv_heads;
    if (groups == 0) return;
    const int start = c0 + h * groups, first = start / share, last = (start + groups - 1) / share;
    if (first == last) return;                                              // finished by its warp
    const PartialView parts(p.scratch, 2 * (size_t)n_warps, p.group, D);
    auto row_of = [&](int gw) -> int64_t {
        return (2 * (int64_t)gw + (gw == first && start != first * share ? 1 : 0)) * p.group + head;
    };
    const int tid = threadIdx.x, nthr = blockDim.x;
    float mx = kNoKey;
    for (int i = first + tid; i <= last; i += nthr) mx = fmaxf(mx, parts.m[row_of(i)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((tid & 31) == 0) s_red[tid >> 5] = mx;
    __syncthreads();
    mx = s_red[0];
    for (int i = 1; i < nthr / 32; i++) mx = fmaxf(mx, s_red[i]);

    const int rp = tid / LPR, lanes = nthr / LPR, d4 = tid % LPR;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int i = first + rp; i <= last; i += lanes) {
        const int64_t r = row_of(i);
        const float f = fast_exp2(parts.m[r] - mx);
        const float4 x = *reinterpret_cast<const float4*>(parts.o + r * D + 4 * d4);
        sum += f * parts.l[r];
        acc.x += f * x.x;
        acc.y += f * x.y;
        acc.z += f * x.z;
        acc.w += f * x.w;
    }
    s_o[tid] = acc;
    if (d4 == 0) s_l[rp] = sum;
    __syncthreads();
    if (rp != 0) return;
    sum = s_l[0];
    for (int i = 1; i < lanes; i++) {
        const float4 x = s_o[i * LPR + d4];
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
        sum += s_l[i];
    }
    if (!(sum != 0.f)) return;                                              // no visible key: the row stays as it is
    const float inv = 1.f / sum;
    uint2 v;
    v.x = Elem<T>::pack2(acc.x * inv, acc.y * inv);
    v.y = Elem<T>::pack2(acc.z * inv, acc.w * inv);
    T* dst = reinterpret_cast<T*>(p.out) + (((int64_t)b * p.num_kv_heads + h) * p.group + head) * D + 4 * d4;
    *reinterpret_cast<uint2*>(dst) = v;
}

template <bool POOL8, typename T, int D, int NQ, bool LIST>
cudaError_t launch_one(const AttendPagesParams& p, int num_sms, cudaStream_t stream) {
    using R = Ring<POOL8, D>;
    constexpr int SLOT = 2 * 16 * D * (POOL8 ? 1 : 2) + (POOL8 ? 32 : 0);
    constexpr size_t ring = (size_t)R::kWarps * R::kStages * SLOT;
    const size_t smem = ring + ((size_t)p.n_seq + 1) * sizeof(int);
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(attend_pages_kernel<POOL8, T, D, NQ, LIST>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)(ring + (kMaxDecodeSeqs + 1) * sizeof(int)));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    e = launch_pdl(attend_pages_kernel<POOL8, T, D, NQ, LIST>, dim3(num_sms), dim3(R::kWarps * 32), smem, stream, p);
    if (e != cudaSuccess) return e;
    // many pieces a pair (few pairs): more threads share a row's merge
    const int n_warps = num_sms * R::kWarps;
    const bool wide = (int64_t)p.n_seq * p.num_kv_heads * 16 < n_warps;
    return launch_pdl(merge_pieces_kernel<T, D>, dim3(p.group * p.num_kv_heads, p.n_seq), dim3(wide ? 512 : 128), 0, stream, p, n_warps);
}

template <typename T, int D, int NQ>
cudaError_t launch_pool(const AttendPagesParams& p, bool pool8, int num_sms, cudaStream_t stream) {
    if (pool8) return p.list ? launch_one<true, T, D, NQ, true>(p, num_sms, stream) : launch_one<true, T, D, NQ, false>(p, num_sms, stream);
    // every page of a 16-bit pool is attend_decode_kernel's work
    return p.list ? launch_one<false, T, D, NQ, true>(p, num_sms, stream) : cudaErrorInvalidValue;
}
template <typename T, int D>
cudaError_t launch_group(const AttendPagesParams& p, bool pool8, int num_sms, cudaStream_t stream) {
    return p.group > 8 ? launch_pool<T, D, 2>(p, pool8, num_sms, stream) : launch_pool<T, D, 1>(p, pool8, num_sms, stream);
}

}  // namespace

size_t attend_pages_scratch_bytes(int group, int head_dim, int num_sms) {
    const size_t slots = 2 * (size_t)num_sms * 16;                          // at most 16 warps an SM
    return (kSplitFloats + slots * group * (head_dim + 2)) * sizeof(float);
}

cudaError_t launch_attend_pages(const AttendPagesParams& p, bool pool8, int head_dim, int dtype, int num_sms, cudaStream_t stream) {
    if (p.n_seq <= 0 || p.max_kv_len <= 0) return cudaSuccess;
    if (p.n_seq > kMaxDecodeSeqs || p.group < 1 || p.group > 16 || p.page_size % 16 != 0) return cudaErrorInvalidValue;
    const bool f16 = dtype == DRKV_DTYPE_F16;
    switch (head_dim) {
        case 64: return f16 ? launch_group<__half, 64>(p, pool8, num_sms, stream) : launch_group<__nv_bfloat16, 64>(p, pool8, num_sms, stream);
        case 128: return f16 ? launch_group<__half, 128>(p, pool8, num_sms, stream) : launch_group<__nv_bfloat16, 128>(p, pool8, num_sms, stream);
        case 256: return f16 ? launch_group<__half, 256>(p, pool8, num_sms, stream) : launch_group<__nv_bfloat16, 256>(p, pool8, num_sms, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace drkv
