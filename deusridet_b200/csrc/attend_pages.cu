// attend_pages.cu — decode attention over the 8-bit pool, and over a list of pages per KV head (either pool).
//
//   o_h = sum_j softmax_j(scale q_h . k_j) v_j       over the keys of the sequence, or of the listed pages only
// The bytes are the cost: (D + 1) per K or V row of the 8-bit pool, 2 D of the 16-bit one, each read once per KV head; the
// 4 D flops per key and query head ride on mma.sync tiles far from their limit (a GQA group fills one 8-column tile).
//
// Split: the keys of all (sequence, KV head) pairs form one line of 16-key groups.  Every warp of a persistent grid takes
// an equal stretch of it, whatever the lengths are: ragged batches need no queue and no tail, and short lines are spread as
// far as they go (1500 keys of 4 heads: 10.4 us a step with one group a warp, 13.5 with four).  A pair that lies inside one
// stretch is finished by its warp; one that is cut leaves a piece (m, l, E, o) per stretch, at most two a warp, and a second
// small kernel merges them in a fixed order (results do not depend on timing).  Warps of one CTA take stretches far apart,
// so that a short line still spreads over all SMs.  Merging inside the kernel, by CTA and then by the last CTA to arrive, took
// 9 us longer on 131 000 keys: fences and a chain of loads by a few CTAs at the end (not measured on short lines).
// Bound by HBM: from 131 001 to 524 001 keys of 8 heads of 128 a key more costs its bytes at 6.1 to 6.4 TB/s (54 and 183 us with
// the merge; at 5.7 in a loop of seconds, where the power cap leaves 1.6 GHz), beside a fixed 10 us for the first data, the
// uneven finish and the merge.  64 sequences of 1-8 k keys, 602 MB: 106 us, 5.7 TB/s.
//
// A warp brings its groups into a private ring of shared memory by cp.async (16 bytes a lane, L1 bypassed), kStages - 1
// groups ahead, and reads them as matrix operands without ldmatrix: contraction order is free, so a lane takes whole
// 16-byte chunks of a row.  Tokens are the M dimension, S^T = K Q^T (A = K rows, B = the group's queries, 8 columns) and
// O^T = V^T P^T (A = V^T, two keys' bytes interleaved by prmt): half the tiles of the usual orientation, where 16 query
// rows would be half empty.  P turns from the accumulator layout into the operand layout by movmatrix.  e4m3 operands
// become f16 two at a time (cvt.rn.f16x2.e4m3x2, exact).
//
// Scales of the 8-bit rows stay exponents.  K's multiply the score.  V's join the weight: what a key adds to o is
// 2^(s + ev) times its bytes (s in the log2 domain), and f16 has 40 binades for the weights of all keys.  So weights have a
// reference of their own beside the softmax's maximum m, per head: E such that m + E is the largest s + ev seen so far.  They
// are 2^((s - m) + (ev - E) + 7), at most 2^15 since they may pass the reference by 2^8 before it follows, of full precision
// down to 2^-20 of the largest, and vanish below 2^-31 of it: next to what the same head has summed, whatever the sizes of
// rows that hold no weight.  o carries 2^E, in the pieces too; the sum of the weights stays relative to m, in fp32.
// (A second exponential and two additions per key and head, measured with one term of P: 64 sequences, 108 us a step with
// them and 109 without; of heads of 64 dims, where a group is half as long, 67 and 66.)
// bf16 queries are scaled by a power of two per head into f16 (8 significant bits fit; exact unless an element is below
// 2^-30 of its row's maximum).  Scores, maxima, sums and outputs accumulate in fp32.
// P in the PV product: f16 hi + lo terms (22 bits) over an 8-bit or an f16 pool, bf16 hi + lo (16 bits) over a bf16 pool.  Only
// bf16 outputs of groups beyond eight heads over the 8-bit pool have one f16 term (2^-12 of a weight beside the output's 2^-9):
// with two column tiles the products count, and 64 sequences of 128 heads take 156 us with two terms, 139 with one.  (Of 32
// heads 113 and 108, of 64 dims 70 and 67, in a loop of seconds, at the 1.65 GHz that the power cap leaves; in a short one, at
// full clock, 108 either way.)
#include <atomic>

#include "kernels.hpp"
#include "kv_common.cuh"
#include "row_tiles.cuh"
#include "sm100_primitives.cuh"

namespace drkv {

namespace {

constexpr float kNoKey = -3.402823466e38f;   // running maximum before any key: no finite score is below it

// Warps per CTA (one CTA per SM) and groups in a warp's ring.
template <bool POOL8, int D, int NQ> struct Ring;
template <int NQ> struct Ring<true, 64, NQ>   { static constexpr int kWarps = 16, kStages = 4; };   // 132 KB
template <> struct Ring<true, 128, 1>         { static constexpr int kWarps = 12, kStages = 4; };   // 198 KB
template <> struct Ring<true, 128, 2>         { static constexpr int kWarps = 12, kStages = 4; };   // 198 KB
template <int NQ> struct Ring<true, 256, NQ>  { static constexpr int kWarps = 8, kStages = 3; };    // 197 KB
template <int NQ> struct Ring<false, 64, NQ>  { static constexpr int kWarps = 16, kStages = 3; };   // 192 KB
template <int NQ> struct Ring<false, 128, NQ> { static constexpr int kWarps = 8, kStages = 3; };    // 192 KB
template <int NQ> struct Ring<false, 256, NQ> { static constexpr int kWarps = 6, kStages = 2; };    // 192 KB

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// An exponent byte that is no less than x; 2^(byte - 127) is finite.
__device__ __forceinline__ float whole_byte(float x) { return fminf(fmaxf(ceilf(x), 0.f), 254.f); }

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

// What the first kernel leaves for the second, in front of the pieces.
struct Split {
    int share, pad[3];
    int cum[kMaxPagesSeqs + 4];        // prefix sums of the line over the sequences
};
constexpr size_t kSplitFloats = sizeof(Split) / 4;

// Pieces: slot = 2 * warp + (the stretch begins inside the pair ? 0 : 1), row = slot * group + head of the group;
// un-normalised sums [row][D], then (maximum in the log2 domain, sum of weights, exponent byte that o is relative to, 0) [row].
struct Pieces {
    float* o;
    float4* mle;
    __host__ __device__ Pieces(float* scratch, int n_warps, int group, int d) {
        o = scratch + kSplitFloats;
        mle = reinterpret_cast<float4*>(o + 2 * (size_t)n_warps * group * d);
    }
};

// Groups of a pair of a sequence.  A list has at most as many entries as the sequence has pages.
__device__ __forceinline__ int pair_groups(const AttendPagesParams& p, int len, bool list) {
    if (len <= 0) return 0;
    if (!list) return (len + 15) >> 4;
    const int pages = (len - 1) / p.page_size + 1;
    return min(pages, p.list_len) * (p.page_size >> 4);
}

// One group of the line as its warp needs it; a warp keeps the next 64 in shared memory.
struct alignas(16) Group {
    int pair, valid;                   // visible keys (0: nothing to read)
    int page, row;                     // pool page; first row in its plane
};

template <bool POOL8, typename T, int D, int NQ, bool LIST>
__global__ void __launch_bounds__(Ring<POOL8, D, NQ>::kWarps * 32, 1) attend_pages_kernel(const AttendPagesParams p) {
    constexpr int WARPS = Ring<POOL8, D, NQ>::kWarps, STAGES = Ring<POOL8, D, NQ>::kStages, THREADS = WARPS * 32;
    using TM = typename std::conditional<POOL8, __half, T>::type;           // matrix operand type
    constexpr bool F16 = std::is_same<TM, __half>::value;
    constexpr bool LO = !(POOL8 && std::is_same<T, __nv_bfloat16>::value && NQ == 2);
    constexpr int ROWB = D * (POOL8 ? 1 : 2), CPR = ROWB / 16, TILE = 16 * ROWB;
    constexpr int SLOT = 2 * TILE + (POOL8 ? 32 : 0);
    constexpr int KSTEPS = D / 16, MT = D / 16;
    constexpr int KCH = CPR / 4;                                            // K chunks a lane reads of a row
    constexpr int EPL = POOL8 ? (D == 64 ? 8 : 16) : 8;                     // V elements a lane reads of a row at once
    constexpr int VCH = D / (8 * EPL);
    // Weights carry 2^WS and may exceed their maximum's by 2^kSlack before the maximum follows: at most 2^15 in f16.
    constexpr float kSlack = 8.f;
    constexpr int WS = F16 ? 7 : 0;
    constexpr uint32_t FULL = 0xffffffffu;

    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_warp_tot[WARPS];
    __shared__ Group s_groups[WARPS][64];
    int* cum = reinterpret_cast<int*>(smem + WARPS * STAGES * SLOT);        // [n_seq + 1]
    int* s_len = cum + p.n_seq + 1;                                         // [n_seq] keys, 0 where nothing is read
    int* s_row = s_len + p.n_seq;                                           // [n_seq] table rows

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    // Lengths, rows and tables were written further back than the kernel directly in front (attend_decode_kernel has the
    // same rule): the split and the first page ids are worked out under that kernel's tail.  A page list may be its output.

    // ---- prefix sums of the line over the sequences ----
    {
        const int per = (p.n_seq + THREADS - 1) / THREADS;
        const int lo = min(tid * per, p.n_seq), hi = min(lo + per, p.n_seq);
        int local = 0;
        for (int b = lo; b < hi; b++) {
            const int row = __ldg(p.rows + b), len = min(__ldg(p.kv_len + b), p.max_kv_len);
            s_row[b] = row;
            s_len[b] = row >= 0 && row < p.max_rows ? len : 0;
            local += pair_groups(p, s_len[b], LIST) * p.num_kv_heads;
        }
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
            run += pair_groups(p, s_len[b], LIST) * p.num_kv_heads;
        }
        if (tid == THREADS - 1) cum[p.n_seq] = run;
        __syncthreads();
    }
    const int total = cum[p.n_seq], n_warps = (int)gridDim.x * WARPS;
    const int share = max(1, (total + n_warps - 1) / n_warps);
    const int gw = w * (int)gridDim.x + (int)blockIdx.x;
    const int64_t lo64 = (int64_t)gw * share;
    const int lo = lo64 < total ? (int)lo64 : total, n = min(share, total - lo);

    // The pair that holds a group of the line, and where it starts and ends.
    struct Span { int pair, start, end; };
    auto pair_at = [&](int f) -> Span {
        int b = 0, e = p.n_seq;                                             // largest b with cum[b] <= f
        while (e - b > 1) {
            const int mid = (b + e) >> 1;
            if (cum[mid] <= f) b = mid; else e = mid;
        }
        const int groups = (cum[b + 1] - cum[b]) / p.num_kv_heads, h = (f - cum[b]) / groups;
        return Span{b * p.num_kv_heads + h, cum[b] + h * groups, cum[b] + (h + 1) * groups};
    };

    // ---- the groups ahead: lane i works out group (window's first) + i; the look-ups are spread over the window before ----
    int ahead_pair = -1, ahead_in = 0, ahead_logical = -1, ahead_page = -1;
    const int per_page = p.page_size >> 4;
    auto locate_pair = [&](int idx) {                                       // step 1: pair and list entry
        ahead_pair = -1;
        ahead_logical = -1;
        if (idx < n) {
            const Span s = pair_at(lo + idx);
            ahead_pair = s.pair;
            const int i = lo + idx - s.start;
            ahead_logical = i / per_page;
            ahead_in = i - ahead_logical * per_page;
            // (a plain load: the kernel in front may have written the list while this one was already running)
            if (LIST) ahead_logical = p.list[(int64_t)s.pair * p.list_len + ahead_logical];
        }
    };
    auto locate_page = [&]() {                                              // step 2: page
        ahead_page = -1;
        if (ahead_pair >= 0 && ahead_logical >= 0 && ahead_logical < p.table_stride)
            ahead_page = __ldg(p.tables + (int64_t)s_row[ahead_pair / p.num_kv_heads] * p.table_stride + ahead_logical);
    };
    auto locate_done = [&](int idx) {                                       // step 3: into the warp's list
        Group r{ahead_pair, 0, 0, 0};
        if (ahead_page >= p.max_pages) {
            atomicExch(p.error_word, (int)KERR_BAD_PAGE);
            ahead_page = -1;
        }
        if (ahead_page >= 0) {
            const int b = ahead_pair / p.num_kv_heads, h = ahead_pair - b * p.num_kv_heads;
            const int len = s_len[b];
            const int64_t tok = (int64_t)ahead_logical * p.page_size + ahead_in * 16;
            if (tok < len) r.valid = min(16, (int)(len - tok));
            r.page = ahead_page;
            r.row = h * p.page_size + ahead_in * 16;
        }
        s_groups[w][idx & 63] = r;
    };
    if (LIST) {
        pdl_wait();
        pdl_launch_dependents();
    }
    locate_pair(lane);
    locate_page();
    locate_done(lane);
    __syncwarp();
    if (!LIST) {
        pdl_wait();
        pdl_launch_dependents();
    }
    if (blockIdx.x == 0) {
        Split* split = reinterpret_cast<Split*>(p.scratch);
        if (tid == 0) split->share = share;
        for (int b = tid; b <= p.n_seq; b += THREADS) split->cum[b] = cum[b];
    }
    if (n <= 0) return;                                                     // no block-wide barrier below

    const uint32_t ring = smem_u32(smem) + w * STAGES * SLOT;
    const uint8_t* lane_src = p.pool + 16 * lane;
    // a lane's chunks of a tile are 32 apart: c = lane + 32 j, row = c / CPR; in the permuted tile the j part of the row
    // contributes a constant XOR and a constant offset to the lane's own place
    const uint32_t lane_dst = tile_off<ROWB>(lane / CPR, lane % CPR);
    auto issue = [&](int idx) {                                             // requests group idx of the stretch
        const int wl = idx & 31;
        const int nx = (idx & ~31) + 32 + lane;
        if ((idx & ~31) + 32 < n) {                                         // the next window's look-ups
            if (wl == 0) locate_pair(nx);
            if (wl == 8) locate_page();
            if (wl == 16) {
                locate_done(nx);
                __syncwarp();
            }
        }
        const Group gr = s_groups[w][idx & 63];
        if (gr.valid == 0) return;
        const uint32_t dst = ring + (idx % STAGES) * SLOT;
        const int64_t block = gr.page * p.block_bytes;
        const uint8_t* k = lane_src + block + (int64_t)gr.row * ROWB;
        const uint8_t* v = k + p.plane_bytes;
#pragma unroll
        for (int j = 0; j < CPR / 2; j++) {
            const int row_j = 32 * j / CPR;                                 // rows below 16, constant
            const uint32_t flip = tile_off<ROWB>(row_j, 0) & 127u, skip = tile_off<ROWB>(row_j, 0) & ~127u;
            const uint32_t off = (lane_dst ^ flip) + skip;
            if (gr.valid == 16) {
                copy16(dst + off, k + 512 * j);
                copy16(dst + TILE + off, v + 512 * j);
            } else {                                                        // hidden rows are zeros: they meet zero weights
                const bool see = (lane + 32 * j) / CPR < gr.valid;
                copy16_or_zero(dst + off, k + 512 * j, see);
                copy16_or_zero(dst + TILE + off, v + 512 * j, see);
            }
        }
        if (POOL8 && lane < 2)                                              // 16 exponents of K, 16 of V
            copy16(dst + 2 * TILE + 16 * lane, p.pool + block + 2 * p.plane_bytes + lane * p.exp_plane_bytes + gr.row);
    };

    // ---- state of the pair being attended ----
    uint32_t qf[NQ][KSTEPS][2];
    float qs[NQ][2];                                                        // score factor of heads 2t and 2t + 1
    float o[NQ][MT][4], m[NQ][2], l[NQ][2];
    float big_e[NQ][2];                                                     // 8-bit pool: E, an exponent byte
    int cur_pair = -1;

    auto begin_pair = [&](int pair) {
        cur_pair = pair;
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
            big_e[nq][0] = big_e[nq][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) o[nq][mt][0] = o[nq][mt][1] = o[nq][mt][2] = o[nq][mt][3] = 0.f;
        }
    };

    const Pieces pieces(p.scratch, n_warps, p.group, D);
    auto end_pair = [&]() {
        const int b = cur_pair / p.num_kv_heads, h = cur_pair - b * p.num_kv_heads;
        const int groups = (cum[b + 1] - cum[b]) / p.num_kv_heads;
        const int start = cum[b] + h * groups;
        const bool whole = start >= lo && start + groups <= lo + n;
        const int64_t row0 = (2 * (int64_t)gw + (start > lo ? 1 : 0)) * p.group;
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float sum = l[nq][c];
                sum += __shfl_xor_sync(FULL, sum, 4);
                sum += __shfl_xor_sync(FULL, sum, 8);
                sum += __shfl_xor_sync(FULL, sum, 16);
                const int head = nq * 8 + 2 * t + c;
                if (head < p.group) {
                    const float f = (whole ? 1.f / sum : 1.f) * (F16 ? 0x1p-7f : 1.f);
                    const float e = POOL8 ? big_e[nq][c] : 127.f, unit = whole ? exp2_int((int)e - 127) : 1.f;
                    if (!whole && g == 0) pieces.mle[row0 + head] = make_float4(m[nq][c], sum, e, 0.f);
#pragma unroll
                    for (int j = 0; j < VCH; j++) {
                        const int dim = (g + 8 * j) * EPL;
                        float x[EPL];
#pragma unroll
                        for (int i = 0; i < EPL / 2; i++) {
                            x[2 * i] = o[nq][j * (EPL / 2) + i][c] * f * unit;
                            x[2 * i + 1] = o[nq][j * (EPL / 2) + i][2 + c] * f * unit;
                        }
                        if (!whole) {
                            float* dst = pieces.o + (row0 + head) * D + dim;
#pragma unroll
                            for (int i = 0; i < EPL; i += 4)
                                *reinterpret_cast<float4*>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                        } else if (sum != 0.f) {                            // no visible key: the row stays as it is
                            T* dst = reinterpret_cast<T*>(p.out) + (((int64_t)b * p.num_kv_heads + h) * p.group + head) * D + dim;
#pragma unroll
                            for (int i = 0; i < EPL; i += 8) {
                                Vec16 v;
#pragma unroll
                                for (int k = 0; k < 4; k++) v.w[k] = Elem<T>::pack2(x[i + 2 * k], x[i + 2 * k + 1]);
                                stg16(dst + i, v);
                            }
                        }
                    }
                }
            }
    };

    auto attend_group = [&](uint32_t tile, int valid) {
        // ---- scores: tokens g and g + 8, heads 2t and 2t + 1 of every 8-head tile ----
        float s[NQ][4];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) s[nq][0] = s[nq][1] = s[nq][2] = s[nq][3] = 0.f;
        float s2[4] = {0.f, 0.f, 0.f, 0.f};                                 // one tile: two chains of dependent products
#pragma unroll
        for (int i = 0; i < KCH; i++) {
            const uint4 ka = lds128(tile + tile_off<ROWB>(g, t + 4 * i)), kb = lds128(tile + tile_off<ROWB>(g + 8, t + 4 * i));
            const uint32_t a[4] = {ka.x, ka.y, ka.z, ka.w}, b[4] = {kb.x, kb.y, kb.z, kb.w};
            if (POOL8) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t a0, a1, a2, a3;
                    e4m3x4_to_f16x4(a[j], a0, a2);
                    e4m3x4_to_f16x4(b[j], a1, a3);
#pragma unroll
                    for (int nq = 0; nq < NQ; nq++)
                        mma16816<TM>(NQ == 1 && (j & 1) ? s2 : s[nq], a0, a1, a2, a3, qf[nq][(4 * i + j) % KSTEPS][0],
                                     qf[nq][(4 * i + j) % KSTEPS][1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int nq = 0; nq < NQ; nq++)
                        mma16816<TM>(NQ == 1 && (j & 1) ? s2 : s[nq], a[2 * j], b[2 * j], a[2 * j + 1], b[2 * j + 1], qf[nq][(2 * i + j) % KSTEPS][0],
                                     qf[nq][(2 * i + j) % KSTEPS][1]);
            }
        }
        if (NQ == 1) {
#pragma unroll
            for (int k = 0; k < 4; k++) s[0][k] += s2[k];
        }
        // s becomes the score in the log2 domain
        float ev0 = 0.f, ev1 = 0.f, ks0 = 1.f, ks1 = 1.f;
        if (POOL8) {
            ks0 = __uint_as_float(max(lds8(tile + 2 * TILE + g) << 23, 0x00400000u));       // 2^(byte - 127), subnormal for 0
            ks1 = __uint_as_float(max(lds8(tile + 2 * TILE + g + 8) << 23, 0x00400000u));
            // byte + WS: the byte as the lowest bits of 2^23
            ev0 = __uint_as_float(0x4b000000u | lds8(tile + 2 * TILE + 16 + g)) - (8388608.f - WS);
            ev1 = __uint_as_float(0x4b000000u | lds8(tile + 2 * TILE + 24 + g)) - (8388608.f - WS);
        }
        if (valid < 16) {                                                   // what lies behind the last key may be anything
            if (g >= valid) ev0 = ks0 = 0.f;
            if (g + 8 >= valid) ev1 = ks1 = 0.f;
        }
        // The maximum and the weights' reference follow only when a score exceeds one of them by more than the slack, and then
        // in full: most groups need no reduction over the lanes.  (Over the 8-bit pool p goes into a sum in fp32 alone, and
        // may pass its maximum by as much as the weights' exponents show.)
        constexpr float LIMIT = POOL8 ? kSlack + WS : kSlack;
        float t0[NQ][2], t1[NQ][2], y0[NQ][2], y1[NQ][2];                   // binary logarithms of p and, with 2^WS, of the weight
        float over = -INFINITY;
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const float f0 = POOL8 ? ks0 * qs[nq][c] : qs[nq][c], f1 = POOL8 ? ks1 * qs[nq][c] : qs[nq][c];
                // the product is rounded before the maximum is taken off, as the maximum was: of scores beyond 2^27 a fused
                // product's lower half alone could exceed the slack
                s[nq][c] = __fmul_rn(s[nq][c], f0);
                s[nq][2 + c] = __fmul_rn(s[nq][2 + c], f1);
                t0[nq][c] = __fadd_rn(s[nq][c], -m[nq][c]);
                t1[nq][c] = __fadd_rn(s[nq][2 + c], -m[nq][c]);
                over = fmax3(over, t0[nq][c], t1[nq][c]);
                if (POOL8) {
                    y0[nq][c] = t0[nq][c] + (ev0 - big_e[nq][c]);
                    y1[nq][c] = t1[nq][c] + (ev1 - big_e[nq][c]);
                    over = fmax3(over, y0[nq][c], y1[nq][c]);
                }
            }
        if (__any_sync(FULL, over > LIMIT)) {
            auto over_keys = [&](float a, float b) -> float {               // maximum over the group's visible keys
                float x = fmaxf(g < valid ? a : -INFINITY, g + 8 < valid ? b : -INFINITY);
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 4));
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 8));
                return fmaxf(x, __shfl_xor_sync(FULL, x, 16));
            };
#pragma unroll
            for (int nq = 0; nq < NQ; nq++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float x = fmaxf(over_keys(s[nq][c], s[nq][2 + c]), m[nq][c]), down = m[nq][c] - x;
                    const float f = fast_exp2(down);
                    float r = f;
                    if (POOL8) {
                        // whole, so that o's unit stays a power of two; never above the largest exponent byte met
                        const float seen = over_keys((s[nq][c] - x) + ev0, (s[nq][2 + c] - x) + ev1) - WS, old = big_e[nq][c];
                        const float e = whole_byte(fmaxf(seen, down + old));
                        r = fast_exp2(down + (old - e));
                        big_e[nq][c] = e;
                    }
                    m[nq][c] = x;
                    t0[nq][c] = __fadd_rn(s[nq][c], -x);
                    t1[nq][c] = __fadd_rn(s[nq][2 + c], -x);
                    y0[nq][c] = t0[nq][c] + (ev0 - big_e[nq][c]);
                    y1[nq][c] = t1[nq][c] + (ev1 - big_e[nq][c]);
                    l[nq][c] *= f;
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        o[nq][mt][c] *= r;
                        o[nq][mt][2 + c] *= r;
                    }
                }
        }
        // ---- weights: p for the sum, w for the product ----
        uint32_t pf[NQ][2], pl[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            float p0[2], p1[2], w0[2], w1[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                p0[c] = fast_exp2(t0[nq][c]);
                p1[c] = fast_exp2(t1[nq][c]);
                w0[c] = POOL8 ? fast_exp2(y0[nq][c]) : p0[c];
                w1[c] = POOL8 ? fast_exp2(y1[nq][c]) : p1[c];
            }
            if (valid < 16) {
                if (g >= valid) p0[0] = p0[1] = w0[0] = w0[1] = 0.f;
                if (g + 8 >= valid) p1[0] = p1[1] = w1[0] = w1[1] = 0.f;
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                l[nq][c] += p0[c] + p1[c];
                if (!POOL8 && F16) {
                    w0[c] *= 0x1p7f;
                    w1[c] *= 0x1p7f;
                }
            }
            const uint32_t h0 = Elem<TM>::pack2(w0[0], w0[1]), h1 = Elem<TM>::pack2(w1[0], w1[1]);
            pf[nq][0] = transpose8x8(h0);
            pf[nq][1] = transpose8x8(h1);
            if (LO) {
                const float2 a = Elem<TM>::unpack2(h0), b = Elem<TM>::unpack2(h1);
                pl[nq][0] = transpose8x8(Elem<TM>::pack2(w0[0] - a.x, w0[1] - a.y));
                pl[nq][1] = transpose8x8(Elem<TM>::pack2(w1[0] - b.x, w1[1] - b.y));
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
                        uint32_t a0, a1, a2, a3;
                        e4m3x4_to_f16x4(x, a0, a1);
                        e4m3x4_to_f16x4(y, a2, a3);
                        pv(j * (EPL / 2) + 2 * i + half, a0, a1, a2, a3);
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
    // (one place each for the start and the end of a pair: the code is long, and short launches pay for fetching it)
    for (int i = 0; i <= n; i++) {
        const int2 meta = *reinterpret_cast<const int2*>(&s_groups[w][i & 63]);   // pair, visible keys
        if (i == n || meta.x != cur_pair) {
            if (cur_pair >= 0) end_pair();
            if (i == n) break;
            begin_pair(meta.x);                                             // its query rows come while the keys do
        }
        if (i + STAGES - 1 < n) issue(i + STAGES - 1);
        copies_commit();
        copies_wait<STAGES - 1>();
        __syncwarp();
        if (meta.y > 0) attend_group(ring + (i % STAGES) * SLOT, meta.y);
        __syncwarp();                                                       // the slot is free for the next request
    }
    copies_wait<0>();
}

// Merges the pieces of the pairs that were cut.  Sets of lanes share a row (one head of one pair), each taking every
// PARTS-th piece, eight pieces' loads in flight at a time: the kernel is a chain of L2 latencies.  CTA_DIMS == 0: many rows of a
// few pieces, one set a row.  CTA_DIMS > 0: a CTA takes that many of one row with as many sets as fit.
template <typename T, int D, int CTA_DIMS>
__global__ void __launch_bounds__(CTA_DIMS ? 256 : 128, 1) merge_pieces_kernel(const AttendPagesParams p, int n_warps) {
    constexpr bool WIDE = CTA_DIMS > 0;
    constexpr int DIMS = WIDE ? CTA_DIMS : D, LANES = DIMS / 4;
    constexpr int PARTS = WIDE ? 256 / LANES : 1, ROWS = WIDE ? 1 : 128 / LANES;
    __shared__ float4 s_o[WIDE ? PARTS : 1][LANES];
    __shared__ float4 s_mle[WIDE ? PARTS : 1];
    pdl_wait();
    pdl_launch_dependents();
    const Split* split = reinterpret_cast<const Split*>(p.scratch);
    const int set = threadIdx.x / LANES, d4 = threadIdx.x % LANES;
    const int hq = p.num_kv_heads * p.group;
    const int row = WIDE ? blockIdx.x : blockIdx.x * ROWS + set, part = WIDE ? set : 0;
    const bool live = row < p.n_seq * hq;
    const int b = live ? row / hq : 0, h = (live ? row - b * hq : 0) / p.group, head = (live ? row - b * hq : 0) - h * p.group;
    const int share = split->share, c0 = split->cum[b], c1 = split->cum[b + 1];
    const int groups = (c1 - c0) / p.num_kv_heads, start = c0 + h * groups;
    const int first = start / share, n = live && groups > 0 ? (start + groups - 1) / share - first + 1 : 0;
    if (WIDE && n < 2) return;                                              // finished by its warp, or no keys
    const Pieces pieces(p.scratch, n_warps, p.group, D);
    const int64_t step = 2 * p.group, row1 = 2 * (int64_t)first * p.group + head;   // piece i > 0 at row1 + i * step
    const int64_t row0 = row1 + (start != first * share ? p.group : 0);
    const float* o = pieces.o + (WIDE ? blockIdx.y * DIMS : 0) + 4 * d4;
    float m = kNoKey, l = 0.f, e = 0.f;                                     // e: exponent byte that acc is relative to
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n >= 2) {
#pragma unroll 1
        for (int i0 = part; i0 < n; i0 += 8 * PARTS) {
            float4 mle[8], x[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = i0 + k * PARTS;
                const int64_t r = i ? row1 + i * step : row0;
                mle[k] = make_float4(kNoKey, 0.f, 0.f, 0.f);
                x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < n) {
                    mle[k] = __ldcg(pieces.mle + r);
                    x[k] = __ldcg(reinterpret_cast<const float4*>(o + r * D));
                }
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, mle[k].x);
            float e_top = (m - top) + e;
#pragma unroll
            for (int k = 0; k < 8; k++) e_top = fmaxf(e_top, (mle[k].x - top) + mle[k].z);
            e_top = whole_byte(e_top);
            l *= fast_exp2(m - top);
            const float f0 = fast_exp2((m - top) + (e - e_top));
            m = top;
            e = e_top;
            acc.x *= f0, acc.y *= f0, acc.z *= f0, acc.w *= f0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float down = mle[k].x - top, f = fast_exp2(down + (mle[k].z - e_top));   // absent: acc stays, 2^.. * 0
                l += mle[k].y * fast_exp2(down);
                acc.x += x[k].x * f, acc.y += x[k].y * f, acc.z += x[k].z * f, acc.w += x[k].w * f;
            }
        }
    }
    if (WIDE) {
        s_o[set][d4] = acc;
        if (d4 == 0) s_mle[set] = make_float4(m, l, e, 0.f);
        __syncthreads();
        if (threadIdx.x >= (LANES > 32 ? LANES : 32)) return;
        // lane i of every warp left works out set i's factors; the sets are added in their order
        const int lane = threadIdx.x & 31;
        const float4 st = lane < PARTS ? s_mle[lane] : make_float4(kNoKey, 0.f, 0.f, 0.f);
        float top = st.x;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
        const float down = st.x - top;
        float e_top = down + st.z;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) e_top = fmaxf(e_top, __shfl_xor_sync(0xffffffffu, e_top, i));
        e = whole_byte(e_top);
        const float fl = fast_exp2(down), fo = fast_exp2(down + (st.z - e));
        l = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < PARTS; i++) {
            const float f = __shfl_sync(0xffffffffu, fo, i);
            const float4 x = s_o[i][d4];
            l += __shfl_sync(0xffffffffu, st.y, i) * __shfl_sync(0xffffffffu, fl, i);
            acc.x += x.x * f, acc.y += x.y * f, acc.z += x.z * f, acc.w += x.w * f;
        }
        if (set != 0) return;
    } else if (n < 2) {
        return;
    }
    if (!(l != 0.f)) return;                                                // no visible key: the row stays as it is
    const float inv = 1.f / l, unit = exp2_int((int)e - 127);
    uint2 v;
    v.x = Elem<T>::pack2(acc.x * inv * unit, acc.y * inv * unit);
    v.y = Elem<T>::pack2(acc.z * inv * unit, acc.w * inv * unit);
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + (int64_t)row * D + (WIDE ? blockIdx.y * DIMS : 0) + 4 * d4) = v;
}

template <bool POOL8, typename T, int D, int NQ, bool LIST>
cudaError_t launch_one(const AttendPagesParams& p, int num_sms, cudaStream_t stream) {
    using R = Ring<POOL8, D, NQ>;
    constexpr int SLOT = 2 * 16 * D * (POOL8 ? 1 : 2) + (POOL8 ? 32 : 0);
    constexpr size_t ring = (size_t)R::kWarps * R::kStages * SLOT;
    const size_t smem = ring + (3 * (size_t)p.n_seq + 1) * sizeof(int);
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(attend_pages_kernel<POOL8, T, D, NQ, LIST>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)(ring + (3 * kMaxPagesSeqs + 1) * sizeof(int)));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    e = launch_pdl(attend_pages_kernel<POOL8, T, D, NQ, LIST>, dim3(num_sms), dim3(R::kWarps * 32), smem, stream, p);
    if (e != cudaSuccess) return e;
    const int n_warps = num_sms * R::kWarps;
    const int64_t pairs = (int64_t)p.n_seq * p.num_kv_heads, rows = pairs * p.group;
    // About n_warps / pairs pieces a row, eight of which a set of lanes takes at a time: the more pieces, the fewer dims a CTA
    // takes and the more sets it has (60 rows of 118 pieces of 256 dims: 20 us a pass with four sets, 15 with thirty-two), as
    // long as the CTAs are resident in two turns (3 360 rows of 9 pieces of 64 dims, a CTA each: 43 us a pass; eight a CTA: 22).
    const int64_t pieces = n_warps / pairs + 2, most = 4 * (int64_t)num_sms;
    if (pieces > 8 && rows <= most) {
        constexpr int MID = D > 64 ? 64 : D;
        if (pieces > 8 * (1024 / MID) && rows * (D / 32) <= most)
            return launch_pdl(merge_pieces_kernel<T, D, 32>, dim3((unsigned)rows, D / 32), dim3(256), 0, stream, p, n_warps);
        if (pieces > 8 * (1024 / D) && rows * (D / MID) <= most)
            return launch_pdl(merge_pieces_kernel<T, D, MID>, dim3((unsigned)rows, D / MID), dim3(256), 0, stream, p, n_warps);
        return launch_pdl(merge_pieces_kernel<T, D, D>, dim3((unsigned)rows), dim3(256), 0, stream, p, n_warps);
    }
    constexpr int per_cta = 128 / (D / 4);
    return launch_pdl(merge_pieces_kernel<T, D, 0>, dim3((unsigned)((rows + per_cta - 1) / per_cta)), dim3(128), 0, stream, p, n_warps);
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
    const size_t rows = 2 * (size_t)num_sms * 16 * group;                  // at most 16 warps a CTA
    return (kSplitFloats + rows * (head_dim + 4)) * sizeof(float);
}

cudaError_t launch_attend_pages(const AttendPagesParams& p, bool pool8, int head_dim, int dtype, int num_sms, cudaStream_t stream) {
    if (p.n_seq <= 0 || p.max_kv_len <= 0) return cudaSuccess;
    if (p.n_seq > kMaxPagesSeqs || p.group < 1 || p.group > 16 || p.page_size % 16 != 0) return cudaErrorInvalidValue;
    const bool f16 = dtype == DRKV_DTYPE_F16;
    switch (head_dim) {
        case 64: return f16 ? launch_group<__half, 64>(p, pool8, num_sms, stream) : launch_group<__nv_bfloat16, 64>(p, pool8, num_sms, stream);
        case 128: return f16 ? launch_group<__half, 128>(p, pool8, num_sms, stream) : launch_group<__nv_bfloat16, 128>(p, pool8, num_sms, stream);
        case 256: return f16 ? launch_group<__half, 256>(p, pool8, num_sms, stream) : launch_group<__nv_bfloat16, 256>(p, pool8, num_sms, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace drkv
