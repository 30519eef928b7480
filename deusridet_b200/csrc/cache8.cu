// cache8.cu — the 8-bit K/V pool: rows quantised as they are written, and read back flat or as a 16-bit image.
//
// A row is one token's K or V of one KV head, x[D].  e = smallest integer with max|x| <= 448 * 2^e, stored
// q = rn_e4m3(x * 2^-e) and the byte e + 127; it stands for q * 2^e.  e4m3 is a floating format, so a power-of-two scale
// costs no precision against amax / 448 (only the subnormal floor moves, to 2^-9 * 2^e, 2^-17 of the row's maximum at
// worst), and scaling by it is exact: each element is rounded ONCE, whoever computes it, and the attention folds the
// scales into exponents.  Non-finite elements do not count towards the maximum; infinities saturate, NaN stays NaN.
// A rotated K row is quantised from its fp32 rotation, not from a 16-bit rounding of it.
// All kernels here are pure data movement (HBM-bound for chunks, launch-bound for decode batches): D / 8 lanes per row, D / 16
// with two runs each in the append, 16-byte vectors on the 16-bit side and 8-byte ones on the 8-bit side, maxima by warp
// shuffle.
#include "kernels.hpp"
#include "kv_common.cuh"
#include "sm100_primitives.cuh"

namespace drkv {

namespace {

constexpr int kThreads8 = 256;
constexpr int kMaxTokens8 = 128;  // tokens of one CTA of the append
constexpr int kBatch8 = 4;        // rows a lane has in flight

// Quantises the row of which each of its LANES lanes holds NV runs of 8 elements, runs l, l + LANES ...; row: its index in the
// block's rows (K plane, then V plane, exponents in the same order).
template <int LANES, int NV>
__device__ __forceinline__ void quantise_row(const float (&x)[8 * NV], uint8_t* block, int64_t exponents, int row, int l, bool store) {
    // the maximum of |x|; NaN is passed over by the maximum, an infinity makes the row look again
    float top = fmaxf(fabsf(x[0]), fabsf(x[1]));
#pragma unroll
    for (int i = 2; i < 8 * NV; i += 2) top = fmax3(top, fabsf(x[i]), fabsf(x[i + 1]));
    uint32_t amax = __float_as_uint(top == top ? top : 0.f);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (__any_sync(0xffffffffu, amax >= 0x7f800000u)) {
        amax = 0;
#pragma unroll
        for (int i = 0; i < 8 * NV; i++) {
            const uint32_t a = __float_as_uint(x[i]) & 0x7fffffffu;
            amax = max(amax, a < 0x7f800000u ? a : 0u);
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    const int e = e4m3_row_exponent(amax);
    const float inv = exp2_int(-e);
    if (!store) return;
    uint8_t* to = block + (int64_t)row * (8 * LANES * NV) + 8 * l;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const float* y = x + 8 * v;
        uint2 q;
        q.x = f32x4_to_e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        q.y = f32x4_to_e4m3x4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
        *reinterpret_cast<uint2*>(to + 8 * LANES * v) = q;
    }
    if (l == 0) block[exponents + row] = (uint8_t)(e + 127);
}

template <typename T>
__device__ __forceinline__ void unpack8(const Vec16& v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = Elem<T>::unpack2(v.w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// 8 stored elements as 16-bit ones: exact, 4 significant bits that came from the type's range, but for fp16's two ends.  A
// row above 64 512 may have rounded up past the largest value and reads as that, and a rotated row's elements may lie
// between the type's steps of 2^-24 and are rounded to the nearest.
template <typename T>
__device__ __forceinline__ Vec16 expand8(uint2 q, int exp_byte) {
    const int e = exp_byte - 127;
    uint32_t h[4];
    e4m3x4_to_f16x4(q.x, h[0], h[1]);
    e4m3x4_to_f16x4(q.y, h[2], h[3]);
    Vec16 v;
    if (Elem<T>::kUmmaFormat == 0 && e >= -14 && e <= 7) {           // within fp16's normal powers and below its end
        const __half2 scale = __half2half2(__ushort_as_half((unsigned short)((e + 15) << 10)));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), scale);
            v.w[i] = *reinterpret_cast<const uint32_t*>(&y);
        }
        return v;
    }
    const float scale = exp2_int(e);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = Elem<__half>::unpack2(h[i]);
        float a = f.x * scale, b = f.y * scale;
        if (Elem<T>::kUmmaFormat == 0) {
            a = fabsf(a) > 65504.f ? copysignf(65504.f, a) : a;      // NaN compares false
            b = fabsf(b) > 65504.f ? copysignf(65504.f, b) : b;
        }
        v.w[i] = Elem<T>::pack2(a, b);
    }
    return v;
}

// Where a CTA's tokens lie: block start (bytes; < 0: hole or no position) and slot.
struct TokenPlace {
    int64_t block;
    int slot, pos;
};

// A CTA takes some tokens, D / 16 lanes per row, two runs of 8 elements a lane: a token's K heads, then its V heads, as in its
// page block.  The next row is on its way while one is worked on.  30 001 tokens of 4 heads of 256 take 33 us, 5.6 TB/s, with half
// of the issue slots and of DRAM's cycles busy: bound by the chain through a row's maximum.  One run a lane (more steps in that chain
// a byte) 41 us, and without the read ahead, a token a CTA, 77.  With the engine's own rotation of K (all 256 dims: angles in fp64,
// a partner's run by shuffle) 62 us; 4 097 tokens of 8 heads of 128 5.4 us without and 8.9 with; 64 tokens 1.9 and 2.5.
constexpr int kAppendRuns = 2;
struct RowRuns { Vec16 v[kAppendRuns]; };
template <typename T, int D>
__global__ void __launch_bounds__(kThreads8, 4) append8_kernel(const Append8Params p, int n_all, int tokens_per_cta, uint32_t magic_rows) {
    constexpr int NV = kAppendRuns, LANES = D / (8 * NV), ROWS = kThreads8 / LANES;
    extern __shared__ float s_trig[];                                // [token][2][half]
    __shared__ TokenPlace s_place[kMaxTokens8];
    pdl_wait();
    pdl_launch_dependents();
    const int tok0 = blockIdx.x * tokens_per_cta, n_tok = min(tokens_per_cta, n_all - tok0);
    const int P = p.layout.page_size, H = p.layout.num_kv_heads;
    const int l = threadIdx.x % LANES, total = n_tok * 2 * H;
    const int64_t exponents = 2 * p.layout.plane;
    auto read = [&](int r) -> RowRuns {
        RowRuns x{};
        if (r >= total) return x;
        const int t = div_magic(r, magic_rows), kh = r - t * 2 * H;
        const T* src = reinterpret_cast<const T*>(kh < H ? p.k_src : p.v_src) + ((int64_t)(tok0 + t) * H + (kh < H ? kh : kh - H)) * D;
#pragma unroll
        for (int v = 0; v < NV; v++) x.v[v] = ldg16(src + 8 * (l + v * LANES));
        return x;
    };
    const int r_own = threadIdx.x / LANES;
    RowRuns a = read(r_own), b;                                      // on its way while the places are worked out
    if (threadIdx.x < n_tok) {
        const int tok = tok0 + threadIdx.x;
        int row = p.row, pos = p.pos_start + tok;
        if (p.rows != nullptr) {
            row = __ldg(p.rows + tok);
            pos = __ldg(p.pos + tok) + p.pos_start;                  // -1 where the lengths count the new token
        }
        const int logical = pos >= 0 ? pos / P : 0;
        int page = -1;
        if (pos >= 0 && logical < p.table_stride && row >= 0 && row < p.max_rows)
            page = __ldg(p.tables + (int64_t)row * p.table_stride + logical);
        const bool live = page >= 0 && page < p.layout.max_pages;    // hole or no position: nothing to write into
        s_place[threadIdx.x] = TokenPlace{live ? p.layout.block_of(p.layer, page) : -1, pos - logical * P, pos};
    }
    __syncthreads();
    const int half = p.rotary_dim >> 1;
    if (half > 0) {
        for (int i = threadIdx.x; i < n_tok * half; i += kThreads8) {   // the angles of append_rope_kernel, bit for bit
            const int t = i / half, j = i - t * half;
            sincos_det(__fmul_rn((float)s_place[t].pos, __ldg(p.inv_freq + j)), s_trig[(2 * t + 1) * half + j], s_trig[2 * t * half + j]);
        }
        __syncthreads();
    }
    auto write = [&](const RowRuns& in, int r) {
        const int t = div_magic(min(r, total - 1), magic_rows), kh = min(r, total - 1) - t * 2 * H;
        float x[8 * NV];
#pragma unroll
        for (int v = 0; v < NV; v++) unpack8<T>(in.v[v], x + 8 * v);
        if (half > 0 && __any_sync(0xffffffffu, kh < H)) {
            const int hl = half / 8;                                 // runs of one rotated half (rotary_dim % 16 == 0)
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int run = l + v * LANES;
                const bool first = run < hl, second = run >= hl && run < 2 * hl;
                const int other = first ? run + hl : second ? run - hl : run;
                // a shuffle within the row's lanes: LANES divides 32 and rows are aligned groups of lanes
                const int from = (threadIdx.x & 31) - l + other % LANES;
                float o[8];
                Vec16 partner;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    partner.w[i] = __shfl_sync(0xffffffffu, in.v[0].w[i], from);
#pragma unroll
                    for (int u = 1; u < NV; u++) {
                        const uint32_t w = __shfl_sync(0xffffffffu, in.v[u].w[i], from);
                        if (other / LANES == u) partner.w[i] = w;
                    }
                }
                unpack8<T>(partner, o);
                if (kh < H && (first || second)) {
                    const float* c = s_trig + 2 * t * half + 8 * (first ? run : run - hl);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        float y0, y1, &mine = x[8 * v + i];
                        rope_pair(first ? mine : o[i], first ? o[i] : mine, c[i], c[half + i], y0, y1);
                        mine = first ? y0 : y1;
                    }
                }
            }
        }
        const TokenPlace at = s_place[t];
        quantise_row<LANES, NV>(x, p.pool + at.block, exponents, kh * P + at.slot, l, r < total && at.block >= 0);
    };
    for (int r0 = 0; r0 < total; r0 += 2 * ROWS) {                   // the whole CTA together: rows r0 + r_own, then the next
        b = read(r0 + ROWS + r_own);
        write(a, r0 + r_own);
        if (r0 + ROWS >= total) break;
        a = read(r0 + 2 * ROWS + r_own);
        write(b, r0 + ROWS + r_own);
    }
}

// grid (token blocks, layer * 2 + plane): a CTA takes some tokens of one plane, four rows a lane at a time.
constexpr int kFlatTokens = 64;   // at most
template <typename T, int D, bool TO_FLAT>
__global__ void __launch_bounds__(kThreads8) flat_copy8_kernel(const Flat8Params p, int tokens_per_cta, uint32_t magic_heads) {
    constexpr int LANES = D / 8, ROWS = kThreads8 / LANES;
    __shared__ TokenPlace s_place[kFlatTokens];
    pdl_wait();
    pdl_launch_dependents();
    const int H = p.layout.num_kv_heads, P = p.layout.page_size;
    const int layer = blockIdx.y >> 1, kv = blockIdx.y & 1;
    const int tok0 = blockIdx.x * tokens_per_cta, n_tok = min(tokens_per_cta, p.num_tokens - tok0);
    if (threadIdx.x < n_tok) {
        const int pos = p.start_token + tok0 + threadIdx.x, logical = pos / P;
        const int page = logical < p.table_stride ? __ldg(p.table + logical) : -1;
        const bool live = page >= 0 && page < p.layout.max_pages;
        s_place[threadIdx.x] = TokenPlace{live ? p.layout.block_of(layer, page) : -1, pos - logical * P, pos};
    }
    __syncthreads();
    const int l = threadIdx.x % LANES, total = n_tok * H;
    const int64_t exponents = 2 * p.layout.plane;
    T* flat = reinterpret_cast<T*>(p.flat) + ((int64_t)blockIdx.y * p.num_tokens + tok0) * H * D + 8 * l;
    for (int r0 = threadIdx.x / LANES; r0 < total + threadIdx.x / LANES; r0 += kBatch8 * ROWS) {   // the whole CTA together
        uint2 q[kBatch8];
        uint8_t e[kBatch8];
        Vec16 in[kBatch8];
#pragma unroll
        for (int u = 0; u < kBatch8; u++) {
            const int r = r0 + u * ROWS;
            q[u] = make_uint2(0u, 0u);
            e[u] = 0;
            in[u] = Vec16{{0u, 0u, 0u, 0u}};
            if (r >= total) continue;
            if (TO_FLAT) {
                const int t = div_magic(r, magic_heads), h = r - t * H;
                const TokenPlace at = s_place[t];
                if (at.block >= 0) {                                 // a hole reads as zeros
                    const uint8_t* block = p.pool + at.block;
                    const int row = (kv * H + h) * P + at.slot;
                    q[u] = __ldcs(reinterpret_cast<const uint2*>(block + (int64_t)row * D) + l);
                    e[u] = block[exponents + row];
                }
            } else {
                in[u] = ldg16(flat + (int64_t)r * D);
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch8; u++) {
            const int r = r0 + u * ROWS;
            if (TO_FLAT) {
                if (r < total) stg16(flat + (int64_t)r * D, expand8<T>(q[u], e[u]));
            } else {
                const int t = div_magic(min(r, total - 1), magic_heads), h = min(r, total - 1) - t * H;
                const TokenPlace at = s_place[t];
                float x[8];
                unpack8<T>(in[u], x);
                quantise_row<LANES, 1>(x, p.pool + at.block, exponents, (kv * H + h) * P + at.slot, l, r < total && at.block >= 0);
            }
        }
    }
}

// 16-bit values with NaN and infinities replaced by zero.
template <typename T>
__device__ __forceinline__ Vec16 finite8(Vec16 v) {
    constexpr uint32_t top = Elem<T>::kUmmaFormat == 0 ? 0x7c00u : 0x7f80u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((v.w[i] & top) == top) v.w[i] &= 0xffff0000u;
        if ((v.w[i] >> 16 & top) == top) v.w[i] &= 0xffffu;
    }
    return v;
}

// grid (logical pages, sequences, parts of a page).  Slots past a sequence's last token may hold anything an earlier owner of
// the page left, and the attention multiplies hidden values by zero: what is not finite there is written as zero.  So of
// several places in tables that name one page the one that sees the most of it has to be the last word: a sequence's last
// page is left to any place that sees more, and of sequences that share the place in their tables the longest writes (the
// later one of equals; this only saves work).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads8) expand8_kernel(const Expand8Params p) {
    constexpr int LANES = D / 8;
    pdl_wait();
    pdl_launch_dependents();
    const int logical = blockIdx.x, s = blockIdx.y, P = p.layout.page_size;
    const int n_tok = p.n_tokens[s];
    if ((int64_t)logical * P >= n_tok || logical >= p.table_stride) return;
    const int page = __ldg(p.tables + (int64_t)p.row[s] * p.table_stride + logical);
    if (page < 0 || page >= p.layout.max_pages) return;
    const int visible = min(P, n_tok - logical * P);
    if (visible < P) {
        int seen = 0;
        for (int o = 0; o < p.n_seq; o++) {
            const int32_t* table = p.tables + (int64_t)p.row[o] * p.table_stride;
            for (int l = threadIdx.x; l < p.table_stride && (int64_t)l * P < p.n_tokens[o]; l += kThreads8)
                seen |= p.n_tokens[o] - l * P > visible && __ldg(table + l) == page;
        }
        if (__syncthreads_or(seen)) return;
    }
    for (int o = 0; o < p.n_seq; o++) {
        if (o == s || (int64_t)logical * P >= p.n_tokens[o]) continue;
        if (p.n_tokens[o] < n_tok || (p.n_tokens[o] == n_tok && o < s)) continue;
        if (__ldg(p.tables + (int64_t)p.row[o] * p.table_stride + logical) == page) return;
    }
    const int rows = 2 * p.layout.num_kv_heads * P;                  // K rows then V rows, exponents in the same order
    const uint8_t* block = p.pool + p.layout.block_of(p.layer, page);
    const uint8_t* exps = block + 2 * p.layout.plane;
    T* image = reinterpret_cast<T*>(p.image) + (int64_t)page * rows * D;
    const int total = rows * LANES;
    for (int i0 = threadIdx.x + blockIdx.z * kBatch8 * kThreads8; i0 < total; i0 += gridDim.z * kBatch8 * kThreads8) {
        uint2 q[kBatch8];
        uint8_t e[kBatch8];
#pragma unroll
        for (int u = 0; u < kBatch8; u++) {
            const int i = i0 + u * kThreads8, r = i / LANES;
            q[u] = make_uint2(0u, 0u);
            e[u] = 0;
            if (i < total) {
                q[u] = __ldcs(reinterpret_cast<const uint2*>(block) + i);
                e[u] = exps[r];                                      // (a plain load: the kernel in front may have written it)
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch8; u++) {
            const int i = i0 + u * kThreads8;
            if (i >= total) continue;
            Vec16 v = expand8<T>(q[u], e[u]);
            if (visible < P && i / LANES % P >= visible) v = finite8<T>(v);
            stg16(image + (int64_t)i * 8, v);
        }
    }
}

// Copy-on-write: a whole page block of every layer (rows past the copied sequence's own are never read).
__global__ void __launch_bounds__(kThreads8) cow_copy8_kernel(const Pool8Layout l, uint8_t* pool, int src_page, int dst_page) {
    pdl_wait();
    pdl_launch_dependents();
    const uint8_t* src = pool + l.block_of(blockIdx.y, src_page);
    uint8_t* dst = pool + l.block_of(blockIdx.y, dst_page);
    for (int64_t i = (int64_t)blockIdx.x * kThreads8 + threadIdx.x; i < l.block / 16; i += (int64_t)gridDim.x * kThreads8)
        stg16(dst + 16 * i, ldg16(src + 16 * i));
}

template <template <typename, int> class Launch, typename P>
cudaError_t by_shape(const P& p, int dtype, int head_dim, int n, int num_sms, cudaStream_t stream) {
    const bool f16 = dtype == DRKV_DTYPE_F16;
    switch (head_dim) {
        case 64: return f16 ? Launch<__half, 64>::run(p, n, num_sms, stream) : Launch<__nv_bfloat16, 64>::run(p, n, num_sms, stream);
        case 128: return f16 ? Launch<__half, 128>::run(p, n, num_sms, stream) : Launch<__nv_bfloat16, 128>::run(p, n, num_sms, stream);
        case 256: return f16 ? Launch<__half, 256>::run(p, n, num_sms, stream) : Launch<__nv_bfloat16, 256>::run(p, n, num_sms, stream);
        default: return cudaErrorInvalidValue;
    }
}
template <typename T, int D>
struct AppendLaunch {
    static cudaError_t run(const Append8Params& p, int n, int num_sms, cudaStream_t s) {
        // A token a CTA for decode batches.  Tokens join while one wave of CTAs is left (4 of 256 threads an SM) until a lane
        // has two rows, the first to work on while the other comes, then up to six while there are two waves; their angles have
        // to fit 32 KB.  (4 097 tokens of 8 heads of 128, written and read: 11.5 us with two rows a lane, 13.0 with one.)
        constexpr int ROWS = kThreads8 / (D / (8 * kAppendRuns));
        const int rows = 2 * p.layout.num_kv_heads, wave = 4 * num_sms;
        int per = 1;
        while (per < kMaxTokens8 && 2 * per * p.rotary_dim <= 8192 &&
               ((per * rows < 2 * ROWS && n >= per * wave) || (per * rows < 6 * ROWS && n >= 2 * per * wave)))
            per *= 2;
        return launch_pdl(append8_kernel<T, D>, dim3((n + per - 1) / per), dim3(kThreads8), (size_t)per * p.rotary_dim * sizeof(float),
                          s, p, n, per, magic_of(rows));
    }
};
// As many tokens a CTA as make one or two batches of rows a lane, fewer while the CTAs do not fill the SMs
// (307 041 tokens of one head of 128 written and read: 83 us so, 110 with 16 a CTA; 1 592 tokens of 5 of 256: 7.8 and 8.4).
template <typename T, int D, bool TO_FLAT>
cudaError_t launch_flat8(const Flat8Params& p, int num_sms, cudaStream_t s) {
    constexpr int ROWS = kThreads8 / (D / 8);
    const int H = p.layout.num_kv_heads;
    int per = kFlatTokens;
    while (per > 1 && per * H >= 2 * kBatch8 * ROWS) per /= 2;
    while (per > 1 && (int64_t)((p.num_tokens + per - 1) / per) * 2 * p.num_layers < 4 * num_sms) per /= 2;
    return launch_pdl(flat_copy8_kernel<T, D, TO_FLAT>, dim3((p.num_tokens + per - 1) / per, 2 * p.num_layers), dim3(kThreads8), 0, s, p, per,
                      magic_of(H));
}
template <typename T, int D>
struct ExtractLaunch {
    static cudaError_t run(const Flat8Params& p, int, int num_sms, cudaStream_t s) { return launch_flat8<T, D, true>(p, num_sms, s); }
};
template <typename T, int D>
struct InjectLaunch {
    static cudaError_t run(const Flat8Params& p, int, int num_sms, cudaStream_t s) { return launch_flat8<T, D, false>(p, num_sms, s); }
};
template <typename T, int D>
struct ExpandLaunch {
    static cudaError_t run(const Expand8Params& p, int n, int num_sms, cudaStream_t s) {
        // Parts of one batch while the CTAs are fewer than two waves of two an SM (one page of 128 tokens of 5 heads of 256: a 43-token chunk takes
        // 51 us in one part, 13 in forty).
        const int batches = (2 * p.layout.num_kv_heads * p.layout.page_size * (D / 8) + kBatch8 * kThreads8 - 1) / (kBatch8 * kThreads8);
        const int parts = min(batches, max(1, 4 * num_sms / (n * p.n_seq)));
        return launch_pdl(expand8_kernel<T, D>, dim3(n, p.n_seq, parts), dim3(kThreads8), 0, s, p);
    }
};

}  // namespace

cudaError_t launch_append8(const Append8Params& p, int n_tokens, int dtype, int num_sms, cudaStream_t stream) {
    if (n_tokens <= 0) return cudaSuccess;
    return by_shape<AppendLaunch>(p, dtype, p.layout.head_dim, n_tokens, num_sms, stream);
}

cudaError_t launch_flat_copy8(const Flat8Params& p, bool to_flat, int dtype, int num_sms, cudaStream_t stream) {
    if (p.num_tokens <= 0) return cudaSuccess;
    if (p.num_layers > 32767) return cudaErrorInvalidValue;          // grid.y
    return to_flat ? by_shape<ExtractLaunch>(p, dtype, p.layout.head_dim, p.num_tokens, num_sms, stream)
                   : by_shape<InjectLaunch>(p, dtype, p.layout.head_dim, p.num_tokens, num_sms, stream);
}

cudaError_t launch_expand8(const Expand8Params& p, int dtype, int num_sms, cudaStream_t stream) {
    int pages = 0;
    for (int i = 0; i < p.n_seq; i++) {
        const int n = (int)(((int64_t)p.n_tokens[i] + p.layout.page_size - 1) / p.layout.page_size);
        pages = n > pages ? n : pages;
    }
    if (pages > p.table_stride) pages = p.table_stride;
    if (pages <= 0) return cudaSuccess;
    return by_shape<ExpandLaunch>(p, dtype, p.layout.head_dim, pages, num_sms, stream);
}

cudaError_t launch_cow_copy8(const Pool8Layout& layout, uint8_t* pool, int src_page, int dst_page, int num_layers, cudaStream_t stream) {
    if (num_layers > 65535) return cudaErrorInvalidValue;
    const int64_t vecs = layout.block / 16;
    const int blocks = (int)((vecs + 4 * kThreads8 - 1) / (4 * kThreads8));
    return launch_pdl(cow_copy8_kernel, dim3(blocks < 64 ? blocks : 64, num_layers), dim3(kThreads8), 0, stream, layout, pool,
                      src_page, dst_page);
}

}  // namespace drkv
