// cache8.cu — the 8-bit K/V pool: rows quantised as they are written, and read back flat or as a 16-bit image.
//
// A row is one token's K or V of one KV head, x[D].  e = smallest integer with max|x| <= 448 * 2^e, stored
// q = rn_e4m3(x * 2^-e) and the byte e + 127; it stands for q * 2^e.  e4m3 is a floating format, so a power-of-two scale
// costs no precision against amax / 448 (only the subnormal floor moves, to 2^-9 * 2^e, 2^-17 of the row's maximum at
// worst), and scaling by it is exact: each element is rounded ONCE, whoever computes it, and the attention folds the
// scales into exponents.  Non-finite elements do not count towards the maximum; infinities saturate, NaN stays NaN.
// A rotated K row is quantised from its fp32 rotation, not from a 16-bit rounding of it.
// All kernels here are pure data movement (HBM-bound for chunks, launch-bound for decode batches): D / 8 lanes per row,
// 16-byte vectors on the 16-bit side and 8-byte ones on the 8-bit side, maxima by warp shuffle.
#include "kernels.hpp"
#include "kv_common.cuh"

namespace drkv {

namespace {

constexpr int kThreads8 = 256;
constexpr int kMaxPairs8 = 128;   // rotary_dim / 2 <= head_dim / 2

// Quantises the row of which each of its LANES lanes holds 8 elements; writes bytes and exponent where store is true.
template <int LANES>
__device__ __forceinline__ void quantise_row(const float (&x)[8], uint8_t* dst, uint8_t* dst_exp, int l, bool store) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t a = __float_as_uint(x[i]) & 0x7fffffffu;
        amax = max(amax, a < 0x7f800000u ? a : 0u);
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const int e = e4m3_row_exponent(amax);
    const float inv = exp2_int(-e);
    uint2 v;
    v.x = f32x2_to_e4m3x2(x[0] * inv, x[1] * inv) | f32x2_to_e4m3x2(x[2] * inv, x[3] * inv) << 16;
    v.y = f32x2_to_e4m3x2(x[4] * inv, x[5] * inv) | f32x2_to_e4m3x2(x[6] * inv, x[7] * inv) << 16;
    if (store) {
        *reinterpret_cast<uint2*>(dst + 8 * l) = v;
        if (l == 0) *dst_exp = (uint8_t)(e + 127);
    }
}

template <typename T>
__device__ __forceinline__ void unpack8(const Vec16& v, float (&x)[8]) {
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
__device__ __forceinline__ Vec16 expand8(uint2 q, float scale) {
    Vec16 v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t two = ((i & 2) ? q.y : q.x) >> (16 * (i & 1));
        const float2 f = Elem<__half>::unpack2(e4m3x2_to_f16x2(two & 0xffffu));
        float a = f.x * scale, b = f.y * scale;
        if (Elem<T>::kUmmaFormat == 0) {
            a = fabsf(a) > 65504.f ? copysignf(65504.f, a) : a;   // NaN compares false
            b = fabsf(b) > 65504.f ? copysignf(65504.f, b) : b;
        }
        v.w[i] = Elem<T>::pack2(a, b);
    }
    return v;
}

// One CTA per token: D / 8 lanes per row, K heads first, then V heads.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads8) append8_kernel(const Append8Params p) {
    constexpr int LANES = D / 8, ROWS = kThreads8 / LANES;
    __shared__ float s_cos[kMaxPairs8], s_sin[kMaxPairs8];
    pdl_wait();
    pdl_launch_dependents();
    const int tok = blockIdx.x;
    int row = p.row, pos = p.pos_start + tok;
    if (p.rows != nullptr) {
        row = __ldg(p.rows + tok);
        pos = __ldg(p.pos + tok) + p.pos_start;                      // -1 where the lengths count the new token
    }
    const int P = p.layout.page_size, H = p.layout.num_kv_heads;
    const int logical = pos >= 0 ? pos / P : 0, slot = pos - logical * P;
    int page = -1;
    if (pos >= 0 && logical < p.table_stride && row >= 0 && row < p.max_rows)
        page = __ldg(p.tables + (int64_t)row * p.table_stride + logical);
    if (page < 0 || page >= p.layout.max_pages) return;             // hole or no position: nothing to write into
    const int half = p.rotary_dim >> 1;
    for (int i = threadIdx.x; i < half; i += kThreads8)              // the angles of append_rope_kernel, bit for bit
        sincos_det(__fmul_rn((float)pos, __ldg(p.inv_freq + i)), s_sin[i], s_cos[i]);
    if (half > 0) __syncthreads();
    const int l = threadIdx.x % LANES;
    uint8_t* block = p.pool + p.layout.block_of(p.layer, page);
    for (int r0 = 0; r0 < 2 * H; r0 += ROWS) {
        const int r = r0 + threadIdx.x / LANES;
        const bool live = r < 2 * H;
        const int kv = r >= H, h = kv ? r - H : r;
        float x[8] = {};
        if (live) {
            const T* src = reinterpret_cast<const T*>(kv ? p.v_src : p.k_src) + ((int64_t)tok * H + h) * D;
            unpack8<T>(ldg16(src + 8 * l), x);
        }
        if (half > 0) {
            const int hl = half / 8;                                 // lanes of one rotated half (rotary_dim % 16 == 0)
            const bool first = l < hl, second = l >= hl && l < 2 * hl;
            // a shuffle within the row's lanes: LANES divides 32 and rows are aligned groups of lanes
            const int base = (threadIdx.x & 31) - l, other = base + (first ? l + hl : second ? l - hl : l);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float o = __shfl_sync(0xffffffffu, x[i], other);
                if (!kv && (first || second)) {
                    const int j = 8 * (first ? l : l - hl) + i;
                    float y0, y1;
                    rope_pair(first ? x[i] : o, first ? o : x[i], s_cos[j], s_sin[j], y0, y1);
                    x[i] = first ? y0 : y1;
                }
            }
        }
        quantise_row<LANES>(x, block + p.layout.row(kv, h, slot), block + p.layout.exponent(kv, h, slot), l, live);
    }
}

// grid (token blocks, layer * 2 + plane): a CTA takes kFlatTokens tokens of one plane.
constexpr int kFlatTokens = 16;
template <typename T, int D, bool TO_FLAT>
__global__ void __launch_bounds__(kThreads8) flat_copy8_kernel(const Flat8Params p) {
    constexpr int LANES = D / 8, ROWS = kThreads8 / LANES;
    pdl_wait();
    pdl_launch_dependents();
    const int H = p.layout.num_kv_heads, P = p.layout.page_size;
    const int layer = blockIdx.y >> 1, kv = blockIdx.y & 1;
    const int tok0 = blockIdx.x * kFlatTokens, n_tok = min(kFlatTokens, p.num_tokens - tok0);
    const int l = threadIdx.x % LANES;
    T* flat = reinterpret_cast<T*>(p.flat) + ((int64_t)blockIdx.y * p.num_tokens + tok0) * H * D;
#pragma unroll 4
    for (int r0 = 0; r0 < n_tok * H; r0 += ROWS) {
        const int r = r0 + threadIdx.x / LANES;
        const bool live = r < n_tok * H;
        const int t = live ? r / H : 0, h = live ? r - t * H : 0;
        const int pos = p.start_token + tok0 + t, logical = pos / P, slot = pos - logical * P;
        int page = logical < p.table_stride ? __ldg(p.table + logical) : -1;
        if (page >= p.layout.max_pages) page = -1;
        uint8_t* block = p.pool + (page < 0 ? 0 : p.layout.block_of(layer, page));
        uint8_t* row = block + p.layout.row(kv, h, slot);
        uint8_t* exponent = block + p.layout.exponent(kv, h, slot);
        T* f = flat + (int64_t)r * D + 8 * l;
        if (TO_FLAT) {
            if (!live) continue;
            Vec16 v = Vec16{{0u, 0u, 0u, 0u}};                       // a hole reads as zeros
            if (page >= 0) v = expand8<T>(*reinterpret_cast<const uint2*>(row + 8 * l), exp2_int((int)*exponent - 127));
            stg16(f, v);
        } else {
            float x[8] = {};
            if (live) unpack8<T>(ldg16(f), x);
            quantise_row<LANES>(x, row, exponent, l, live && page >= 0);
        }
    }
}

// grid (logical pages, sequences).  Of several sequences that share a page the one that sees the most tokens (the later
// one of equals) writes it, so no address has two writers.  Slots past its last token read as zero: what an earlier
// owner of the page left there may be NaN, and the attention multiplies hidden values by zero.
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
    for (int o = 0; o < p.n_seq; o++) {
        if (o == s || (int64_t)logical * P >= p.n_tokens[o]) continue;
        if (p.n_tokens[o] < n_tok || (p.n_tokens[o] == n_tok && o < s)) continue;
        if (__ldg(p.tables + (int64_t)p.row[o] * p.table_stride + logical) == page) return;
    }
    const int visible = min(P, n_tok - logical * P);
    const int rows = 2 * p.layout.num_kv_heads * P;                  // K rows then V rows, exponents in the same order
    const uint8_t* block = p.pool + p.layout.block_of(p.layer, page);
    const uint8_t* exps = block + 2 * p.layout.plane;
    T* image = reinterpret_cast<T*>(p.image) + (int64_t)page * rows * D;
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * LANES; i += kThreads8) {
        const int r = i / LANES;
        Vec16 v = Vec16{{0u, 0u, 0u, 0u}};
        if (r % P < visible)
            v = expand8<T>(__ldg(reinterpret_cast<const uint2*>(block) + i), exp2_int((int)__ldg(exps + r) - 127));
        stg16(image + (int64_t)i * 8, v);
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
cudaError_t by_shape(const P& p, int dtype, int head_dim, int n, cudaStream_t stream) {
    const bool f16 = dtype == DRKV_DTYPE_F16;
    switch (head_dim) {
        case 64: return f16 ? Launch<__half, 64>::run(p, n, stream) : Launch<__nv_bfloat16, 64>::run(p, n, stream);
        case 128: return f16 ? Launch<__half, 128>::run(p, n, stream) : Launch<__nv_bfloat16, 128>::run(p, n, stream);
        case 256: return f16 ? Launch<__half, 256>::run(p, n, stream) : Launch<__nv_bfloat16, 256>::run(p, n, stream);
        default: return cudaErrorInvalidValue;
    }
}
template <typename T, int D>
struct AppendLaunch {
    static cudaError_t run(const Append8Params& p, int n, cudaStream_t s) {
        return launch_pdl(append8_kernel<T, D>, dim3(n), dim3(kThreads8), 0, s, p);
    }
};
template <typename T, int D>
struct ExtractLaunch {
    static cudaError_t run(const Flat8Params& p, int n, cudaStream_t s) {
        return launch_pdl(flat_copy8_kernel<T, D, true>, dim3(n, 2 * p.num_layers), dim3(kThreads8), 0, s, p);
    }
};
template <typename T, int D>
struct InjectLaunch {
    static cudaError_t run(const Flat8Params& p, int n, cudaStream_t s) {
        return launch_pdl(flat_copy8_kernel<T, D, false>, dim3(n, 2 * p.num_layers), dim3(kThreads8), 0, s, p);
    }
};
template <typename T, int D>
struct ExpandLaunch {
    static cudaError_t run(const Expand8Params& p, int n, cudaStream_t s) {
        return launch_pdl(expand8_kernel<T, D>, dim3(n, p.n_seq), dim3(kThreads8), 0, s, p);
    }
};

}  // namespace

cudaError_t launch_append8(const Append8Params& p, int n_tokens, int dtype, cudaStream_t stream) {
    if (n_tokens <= 0) return cudaSuccess;
    return by_shape<AppendLaunch>(p, dtype, p.layout.head_dim, n_tokens, stream);
}

cudaError_t launch_flat_copy8(const Flat8Params& p, bool to_flat, int dtype, cudaStream_t stream) {
    if (p.num_tokens <= 0) return cudaSuccess;
    if (p.num_layers > 32767) return cudaErrorInvalidValue;          // grid.y
    const int blocks = (p.num_tokens + kFlatTokens - 1) / kFlatTokens;
    return to_flat ? by_shape<ExtractLaunch>(p, dtype, p.layout.head_dim, blocks, stream)
                   : by_shape<InjectLaunch>(p, dtype, p.layout.head_dim, blocks, stream);
}

cudaError_t launch_expand8(const Expand8Params& p, int dtype, cudaStream_t stream) {
    int pages = 0;
    for (int i = 0; i < p.n_seq; i++) {
        const int n = (int)(((int64_t)p.n_tokens[i] + p.layout.page_size - 1) / p.layout.page_size);
        pages = n > pages ? n : pages;
    }
    if (pages > p.table_stride) pages = p.table_stride;
    if (pages <= 0) return cudaSuccess;
    return by_shape<ExpandLaunch>(p, dtype, p.layout.head_dim, pages, stream);
}

cudaError_t launch_cow_copy8(const Pool8Layout& layout, uint8_t* pool, int src_page, int dst_page, int num_layers, cudaStream_t stream) {
    if (num_layers > 65535) return cudaErrorInvalidValue;
    const int64_t vecs = layout.block / 16;
    const int blocks = (int)((vecs + 4 * kThreads8 - 1) / (4 * kThreads8));
    return launch_pdl(cow_copy8_kernel, dim3(blocks < 64 ? blocks : 64, num_layers), dim3(kThreads8), 0, stream, layout, pool,
                      src_page, dst_page);
}

}  // namespace drkv
