// rope.cu — rotary positions for query and key rows of any strides, both in one launch.
//
// The engine's append rotates K on its way into the cache (src/machina/layer_attention.cu:32-79: halves layout, no
// scaling, fp32 angles) and leaves Q to the caller.  This operator rotates both, in either layout, over part of the
// head, with the frequency scalings that long contexts use, and its transpose (the gradient).  Pair i of a head:
//   y0 = a (x0 c - x1 s),  y1 = a (x1 c + x0 s),   c, s = cos, sin(pos * f_i)          (transpose: s -> -s)
//   halves: (x0, x1) = (x[i], x[i + rot/2])        pairs: (x0, x1) = (x[2i], x[2i + 1])
// Angles: the host keeps t_i = frac(f_i / 2 pi) * 2^64 as an integer, so pos * t_i mod 2^64 IS the phase, exact to
// 2^-64 of a turn per position however far the position is; its upper 32 bits go to fp32 as half turns for sincospif.
// An fp32 product pos * f_i would be off by up to 0.03 rad at position 10^6.
// Pure data movement: every element is read once and written once (6 flops per pair); HBM-bound for chunks,
// launch-bound for decode batches.
#include <cmath>
#include <cstring>
#include <new>
#include <type_traits>
#include <vector>

#include "device_guard.hpp"
#include "kernels.hpp"
#include "kv_common.cuh"
#include "stateless.hpp"

struct drkv_rope {
    drkv_rope_config cfg{};
    std::vector<double> freq;        // radians per position, per pair
    uint64_t* d_turns = nullptr;     // [rotary_dim / 2]
    float factor = 1.f;
    int num_sms = 148;
};

namespace drkv {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeUnroll = 4;       // items a thread of the general kernel has in flight

struct RopeRowsDev {
    const void* src;
    void* dst;
    int64_t src_token, src_head, dst_token, dst_head;   // strides in elements
};

struct RopeParams {
    RopeRowsDev q, k;
    const int32_t* pos;
    const uint64_t* turns;
    int n_tokens, q_heads, heads;    // heads = query heads + key heads
    int half, rotary_dim, tokens_per_cta, heads_per_cta;
    int pairs_layout, inverse;
    float factor;
    // items of one (token, head) row: rot_items of VW pairs each, then copy_items of VW elements each (rows that
    // are not rotated in place)
    int rot_items, row_items;
    uint32_t magic_row, magic_heads; // of row_items and heads_per_cta, see div_magic
};

// Cosines and sines of a CTA's tokens, one pair per thread: [token][cosines | sines][pad].  PER_DIM: one of each for every
// dim that turns, the sine with the sign that the dim's own formula gives it; a lane's eight as two vectors that stand where
// its neighbours' do not collide (trig_place).
__device__ __forceinline__ int trig_place(int dim, int pad) { return (dim & 4 ? pad / 2 : 0) + (dim >> 3) * 4 + (dim & 3); }
template <bool PER_DIM>
__device__ __forceinline__ void fill_trig(const RopeParams& p, float* s_trig, int tok0, int n_tok, int pad) {
    const int n = PER_DIM ? p.half : pad;
    for (int i = threadIdx.x; i < n_tok * n; i += kRopeThreads) {
        const int t = i / n, j = i - t * n;
        if (j < p.half) {
            const uint64_t phase = (uint64_t)(int64_t)__ldg(p.pos + tok0 + t) * __ldg(p.turns + j);
            const int hi = (int)(uint32_t)((phase + 0x80000000ull) >> 32);
            float s, c;
            sincospif((float)hi * 0x1p-31f, &s, &c);
            c *= p.factor;
            s = (p.inverse ? -s : s) * p.factor;
            float* to = s_trig + t * 2 * pad;
            const int at = PER_DIM ? trig_place(j, pad) : j;
            to[at] = c;
            to[pad + at] = PER_DIM ? -s : s;
            if (PER_DIM) {
                const int beside = trig_place(j + p.half, pad);
                to[beside] = c;
                to[pad + beside] = s;
            }
        }
    }
}

template <int VW> struct RopeVec;
template <> struct RopeVec<8> { using type = uint4; };
template <> struct RopeVec<4> { using type = uint2; };
template <> struct RopeVec<2> { using type = uint32_t; };
template <> struct RopeVec<1> { using type = uint16_t; };

// A thread takes items of VW pairs (two vectors of VW elements).  VW is the widest of 8, 4, 2, 1 that divides half the
// rotated dims and every stride and alignment; 16-byte vectors for the usual heads, 2-byte ones only for odd halves.
// tokens_per_cta tokens share a CTA: their cosines and sines are evaluated once into shared memory, one per thread,
// and used by every head (blockIdx.y: a share of the heads, while there are few tokens).
template <typename T, int VW>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
    extern __shared__ __align__(16) float s_trig[];             // [tokens_per_cta][2][half_pad]
    using V = typename RopeVec<VW>::type;
    pdl_wait();
    pdl_launch_dependents();
    const int half = p.half, pad = (half + 3) & ~3;
    const int tok0 = blockIdx.x * p.tokens_per_cta;
    const int n_tok = min(p.tokens_per_cta, p.n_tokens - tok0);
    fill_trig<false>(p, s_trig, tok0, n_tok, pad);
    __syncthreads();
    const uint32_t per_token = (uint32_t)p.heads_per_cta * p.row_items, total = per_token * n_tok;
    for (uint32_t base = threadIdx.x; base < total; base += kRopeThreads * kRopeUnroll) {
        V a[kRopeUnroll], b[kRopeUnroll];
        T* dst[kRopeUnroll];
        int off_b[kRopeUnroll], trig[kRopeUnroll];              // trig < 0: a copy of one vector; off_b < 0: nothing
#pragma unroll
        for (int u = 0; u < kRopeUnroll; u++) {
            const uint32_t it = base + u * kRopeThreads;
            off_b[u] = -1;
            trig[u] = -1;
            if (it >= total) continue;
            const uint32_t row = div_magic(it, p.magic_row), j = it - row * p.row_items;
            const uint32_t t = div_magic(row, p.magic_heads), h = row - t * p.heads_per_cta + blockIdx.y * p.heads_per_cta;
            if ((int)h >= p.heads) continue;
            const bool is_k = (int)h >= p.q_heads;
            const RopeRowsDev& r = is_k ? p.k : p.q;
            const int64_t head = is_k ? (int)h - p.q_heads : (int)h, tok = tok0 + (int)t;
            const T* src = reinterpret_cast<const T*>(r.src) + tok * r.src_token + head * r.src_head;
            dst[u] = reinterpret_cast<T*>(r.dst) + tok * r.dst_token + head * r.dst_head;
            if ((int)j < p.rot_items) {
                const int first = p.pairs_layout ? 2 * VW * j : VW * j;
                off_b[u] = p.pairs_layout ? VW : half;
                trig[u] = t * 2 * pad + VW * j;
                a[u] = *reinterpret_cast<const V*>(src + first);
                b[u] = *reinterpret_cast<const V*>(src + first + off_b[u]);
                dst[u] += first;
            } else {
                const int first = p.rotary_dim + VW * ((int)j - p.rot_items);
                off_b[u] = 0;
                a[u] = *reinterpret_cast<const V*>(src + first);
                dst[u] += first;
            }
        }
#pragma unroll
        for (int u = 0; u < kRopeUnroll; u++) {
            if (off_b[u] < 0) continue;
            if (trig[u] >= 0) {
                T xa[VW], xb[VW], ya[VW], yb[VW];
                memcpy(xa, &a[u], sizeof(V));
                memcpy(xb, &b[u], sizeof(V));
                const float* c = s_trig + trig[u];
                const float* s = c + pad;
#pragma unroll
                for (int i = 0; i < VW; i++) {
                    // element 2i, 2i + 1 of the 2 VW contiguous ones (pairs), or i of either half
                    const T e0 = p.pairs_layout ? (2 * i < VW ? xa[(2 * i) % VW] : xb[(2 * i) % VW]) : xa[i];
                    const T e1 = p.pairs_layout ? (2 * i + 1 < VW ? xa[(2 * i + 1) % VW] : xb[(2 * i + 1) % VW]) : xb[i];
                    float y0, y1;
                    rope_pair(Elem<T>::to_f(e0), Elem<T>::to_f(e1), c[i], s[i], y0, y1);
                    const T r0 = Elem<T>::from_f(y0), r1 = Elem<T>::from_f(y1);
                    if (p.pairs_layout) {
                        if (2 * i < VW) ya[(2 * i) % VW] = r0; else yb[(2 * i) % VW] = r0;
                        if (2 * i + 1 < VW) ya[(2 * i + 1) % VW] = r1; else yb[(2 * i + 1) % VW] = r1;
                    } else {
                        ya[i] = r0;
                        yb[i] = r1;
                    }
                }
                memcpy(&a[u], ya, sizeof(V));
                memcpy(&b[u], yb, sizeof(V));
                *reinterpret_cast<V*>(dst[u] + off_b[u]) = b[u];
            }
            *reinterpret_cast<V*>(dst[u]) = a[u];
        }
    }
}

// The usual heads (64, 128 or 256 dims, 16-byte vectors): a lane takes one vector of a row, its partners of the other half
// come by shuffle (pairs: they are in the same vector), and the next row is on its way while one is worked on.  32 registers, so
// that 2 048 threads an SM keep loads in flight: 32 768 tokens of 40 heads of 128 122 us (5.5 TB/s); four rows a lane at 80
// registers: 138.
// (The general kernel above loses on them by index arithmetic per vector: 158 us.)
// Halves of a width that is no multiple of 8 (kAnyHalves): a lane's partners lie across two vectors, so a warp lays the row
// into shared memory as a ring (the first half once more behind the second), where the partner of dim e is at e + half
// (50 of 64 dims of 28 heads, 7 401 tokens: 17 us; the general kernel, by single elements, 39.  116 of 128 dims of 36 heads,
// 16 824 tokens: 84 us; by words 104; this with the row read back by words and a lane's cosines side by side 110: shared
// memory's banks are what it is short of).
enum RopeMode { kHalves, kPairs, kAnyHalves };

// Elements of a row's ring: rotary_dim + half, and what a lane reads past its own.
__host__ __device__ constexpr int ring_elements(int lanes) { return 12 * lanes + 16; }

template <typename T, int MODE>
__global__ void __launch_bounds__(kRopeThreads, MODE == kAnyHalves ? 4 : 8) rope_rows_kernel(const RopeParams p, int lanes_log2) {
    constexpr bool PAIRS = MODE == kPairs, ANY = MODE == kAnyHalves;
    extern __shared__ __align__(16) float s_trig[];             // [tokens_per_cta][2][pad], then the rows' rings
    pdl_wait();
    pdl_launch_dependents();
    const int half = p.half, pad = ANY ? (p.rotary_dim + 7) & ~7 : (half + 3) & ~3;
    const int tok0 = blockIdx.x * p.tokens_per_cta, n_tok = min(p.tokens_per_cta, p.n_tokens - tok0);
    const int lanes = 1 << lanes_log2, l = threadIdx.x & (lanes - 1), rows_at_once = kRopeThreads >> lanes_log2;
    const int total = n_tok * p.heads_per_cta, rot_lanes = (p.rotary_dim + 7) >> 3, half_lanes = half >> 3;
    const bool turns = l < rot_lanes;
    const int live_pairs = half - 4 * l;                        // of the lane's four words, those that turn (not kHalves)
    const bool second = !PAIRS && l >= half_lanes;
    const uint32_t flip = second ? 0u : 0x80008000u;            // both signs of a word
    const int partner = (threadIdx.x & 31) + (PAIRS || !turns ? 0 : second ? -half_lanes : half_lanes);
    const int trig0 = !turns ? 0 : PAIRS || ANY ? 4 * l : 8 * (second ? l - half_lanes : l);
    const int ring = ring_elements(lanes);
    uint32_t* row_ring = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(s_trig + p.tokens_per_cta * 2 * pad) + (threadIdx.x >> lanes_log2) * ring);
    struct Row {
        Vec16 v;
        T* dst;                                                 // null: nothing to write
        int tok;
    };
    auto read = [&](int row) -> Row {
        Row x{Vec16{{0u, 0u, 0u, 0u}}, nullptr, 0};
        if (row >= total) return x;
        const int t = div_magic(row, p.magic_heads), h = row + ((int)blockIdx.y - t) * p.heads_per_cta;
        if (h >= p.heads) return x;
        const bool is_k = h >= p.q_heads;
        const RopeRowsDev& r = is_k ? p.k : p.q;
        if (!turns && r.src == r.dst) return x;                 // in place, and these dims stay
        const int64_t head = is_k ? h - p.q_heads : h;
        x.v = ldg16(reinterpret_cast<const T*>(r.src) + (int64_t)(tok0 + t) * r.src_token + head * r.src_head + 8 * l);
        x.dst = reinterpret_cast<T*>(r.dst) + (int64_t)(tok0 + t) * r.dst_token + head * r.dst_head + 8 * l;
        x.tok = t;
        return x;
    };
    auto write = [&](const Row& x) {
        const float4* cs = reinterpret_cast<const float4*>(s_trig + x.tok * 2 * pad + trig0);   // 16-byte aligned: pad % 4 == 0
        float c[8], s[8];
#pragma unroll
        for (int i = 0; i < (PAIRS ? 1 : 2); i++) {
            *reinterpret_cast<float4*>(c + 4 * i) = cs[ANY ? pad / 8 * i : i];
            *reinterpret_cast<float4*>(s + 4 * i) = cs[pad / 4 + (ANY ? pad / 8 * i : i)];
        }
        Vec16 y, other = x.v;
        if (ANY) {
            __syncwarp();                                       // the row before has been read
            if (live_pairs >= 4) *reinterpret_cast<Vec16*>(row_ring + 4 * l) = x.v;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (live_pairs < 4 && i < live_pairs) row_ring[4 * l + i] = x.v.w[i];
                if (8 * l + 2 * i < half) row_ring[half + 4 * l + i] = x.v.w[i];
            }
            __syncwarp();
            if (turns) {
                // the two vectors that hold dims 8 l + half and on, shifted to their first
                const Vec16* from = reinterpret_cast<const Vec16*>(row_ring) + ((8 * l + half) >> 3);
                const Vec16 v0 = from[0], v1 = from[1];
                const uint32_t bits = half & 1 ? 16 : 0;
                auto shifted = [&](auto words) {
                    constexpr int W = decltype(words)::value;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t lo = i + W < 4 ? v0.w[(i + W) & 3] : v1.w[(i + W) & 3];
                        const uint32_t hi = i + W + 1 < 4 ? v0.w[(i + W + 1) & 3] : v1.w[(i + W + 1) & 3];
                        other.w[i] = __funnelshift_r(lo, hi, bits);
                    }
                };
                switch (half >> 1 & 3) {
                    case 0: shifted(std::integral_constant<int, 0>{}); break;
                    case 1: shifted(std::integral_constant<int, 1>{}); break;
                    case 2: shifted(std::integral_constant<int, 2>{}); break;
                    default: shifted(std::integral_constant<int, 3>{}); break;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 own = Elem<T>::unpack2(x.v.w[i]);
            float y0, y1;
            if (PAIRS) {
                rope_pair(own.x, own.y, c[i], s[i], y0, y1);
            } else {
                // first half: x0 c - x1 s; second: x1 c + x0 s (kAnyHalves: the sign is the table's)
                const uint32_t w = ANY ? other.w[i] : __shfl_sync(0xffffffffu, x.v.w[i], partner) ^ flip;
                const float2 o = Elem<T>::unpack2(w);
                y0 = __fmaf_rn(own.x, c[2 * i], __fmul_rn(o.x, s[2 * i]));
                y1 = __fmaf_rn(own.y, c[2 * i + 1], __fmul_rn(o.y, s[2 * i + 1]));
            }
            y.w[i] = (MODE == kHalves ? turns : i < live_pairs) ? Elem<T>::pack2(y0, y1) : x.v.w[i];
        }
        if (x.dst != nullptr) stg16(x.dst, y);
    };
    const int r_own = threadIdx.x >> lanes_log2;
    Row a = read(r_own), b;                                     // on its way while the cosines are evaluated
    fill_trig<ANY>(p, s_trig, tok0, n_tok, pad);
    __syncthreads();
    for (int r0 = 0; r0 < total; r0 += 2 * rows_at_once) {      // the whole CTA together: rows r0 + r_own, then the next
        b = read(r0 + rows_at_once + r_own);
        write(a);
        if (r0 + rows_at_once >= total) break;
        a = read(r0 + 2 * rows_at_once + r_own);
        write(b);
    }
}

int fail(int code, const char* msg) {
    set_last_error(msg);
    return code;
}

// Largest vector width the rows allow: every address they form is a multiple of it.
int widest(const drkv_rope_rows& r, int n_tokens, int vw) {
    auto fits = [&](const void* ptr, int64_t tok, int64_t head) {
        return reinterpret_cast<uintptr_t>(ptr) % (2 * (size_t)vw) == 0 && (n_tokens < 2 || tok % vw == 0) &&
               (r.heads < 2 || head % vw == 0);
    };
    while (vw > 1 && !(fits(r.src, r.src_token_stride, r.src_head_stride) && fits(r.dst, r.dst_token_stride, r.dst_head_stride)))
        vw >>= 1;
    return vw;
}

// Rows of the destination must not overlap one another: the larger of the two strides has to step over what the
// smaller one covers.
bool rows_apart(int64_t tok, int64_t head, int n_tokens, int heads, int d) {
    if (n_tokens < 2) tok = INT64_MAX / 4;
    if (heads < 2) head = INT64_MAX / 4;
    if (tok < 0 || head < 0) return false;
    if (head <= tok) return head >= d && (heads < 2 || n_tokens < 2 || tok >= head * (heads - 1) + d);
    return tok >= d && (heads < 2 || n_tokens < 2 || head >= tok * (n_tokens - 1) + d);
}

template <typename T>
cudaError_t launch_rope(const RopeParams& p, int vw, dim3 grid, size_t smem, cudaStream_t stream) {
    switch (vw) {
        case 8: return launch_pdl(rope_kernel<T, 8>, grid, dim3(kRopeThreads), smem, stream, p);
        case 4: return launch_pdl(rope_kernel<T, 4>, grid, dim3(kRopeThreads), smem, stream, p);
        case 2: return launch_pdl(rope_kernel<T, 2>, grid, dim3(kRopeThreads), smem, stream, p);
        default: return launch_pdl(rope_kernel<T, 1>, grid, dim3(kRopeThreads), smem, stream, p);
    }
}

template <typename T>
cudaError_t launch_rows(const RopeParams& p, int mode, int lg, dim3 grid, size_t smem, cudaStream_t stream) {
    switch (mode) {
        case kPairs: return launch_pdl(rope_rows_kernel<T, kPairs>, grid, dim3(kRopeThreads), smem, stream, p, lg);
        case kHalves: return launch_pdl(rope_rows_kernel<T, kHalves>, grid, dim3(kRopeThreads), smem, stream, p, lg);
        default: return launch_pdl(rope_rows_kernel<T, kAnyHalves>, grid, dim3(kRopeThreads), smem, stream, p, lg);
    }
}

// f_i in radians per position, in extended precision.
void frequencies(const drkv_rope_config& c, std::vector<long double>* out) {
    const long double pi = 3.141592653589793238462643383279502884L;
    const int rot = c.rotary_dim;
    long double theta = c.theta;
    const long double factor = c.factor;
    if (c.scaling == DRKV_ROPE_BASE) theta *= powl(factor, (long double)rot / (rot - 2));
    out->resize(rot / 2);
    long double low = 0, high = 0;
    if (c.scaling == DRKV_ROPE_RAMP) {
        auto pair_of = [&](long double turns) {       // the pair that makes `turns` turns over the original context
            return rot * logl(c.original_context / (turns * 2 * pi)) / (2 * logl(theta));
        };
        low = floorl(pair_of(c.beta_fast));
        high = ceill(pair_of(c.beta_slow));
        if (low < 0) low = 0;
        if (high > rot - 1) high = rot - 1;
    }
    for (int i = 0; i < rot / 2; i++) {
        long double f = powl(theta, -2.0L * i / rot);
        if (c.scaling == DRKV_ROPE_LINEAR) f /= factor;
        if (c.scaling == DRKV_ROPE_BANDS) {
            const long double turns = c.original_context * f / (2 * pi);
            long double keep = (turns - c.low_freq_factor) / ((long double)c.high_freq_factor - c.low_freq_factor);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * ((1 - keep) / factor + keep);
        }
        if (c.scaling == DRKV_ROPE_RAMP) {
            const long double width = high - low > 0.001L ? high - low : 0.001L;
            long double r = (i - low) / width;
            r = r < 0 ? 0 : r > 1 ? 1 : r;
            f = f / factor * r + f * (1 - r);
        }
        (*out)[i] = f;
    }
}

}  // namespace

}  // namespace drkv

using namespace drkv;

extern "C" {

int drkv_rope_create(const drkv_rope_config* cfg, drkv_rope** out) {
    if (!cfg || !out) return fail(DRKV_ERR_INVALID, "rope_create: null argument");
    *out = nullptr;
    const drkv_rope_config& c = *cfg;
    if (c.head_dim < 8 || c.head_dim > 512 || c.head_dim % 8 != 0)
        return fail(DRKV_ERR_INVALID, "rope_create: head_dim must be a multiple of 8 up to 512");
    if (c.rotary_dim < 2 || c.rotary_dim > c.head_dim || c.rotary_dim % 2 != 0)
        return fail(DRKV_ERR_INVALID, "rope_create: rotary_dim must be even, positive and within head_dim");
    if (c.dtype != DRKV_DTYPE_F16 && c.dtype != DRKV_DTYPE_BF16)
        return fail(DRKV_ERR_INVALID, "rope_create: dtype must be f16 or bf16");
    if (c.layout != DRKV_ROPE_HALVES && c.layout != DRKV_ROPE_PAIRS)
        return fail(DRKV_ERR_INVALID, "rope_create: unknown layout");
    if (c.scaling < DRKV_ROPE_NONE || c.scaling > DRKV_ROPE_RAMP) return fail(DRKV_ERR_INVALID, "rope_create: unknown scaling");
    if (!(c.theta > 1.0) || !std::isfinite(c.theta)) return fail(DRKV_ERR_INVALID, "rope_create: theta must be above 1");
    if (c.scaling != DRKV_ROPE_NONE && (!(c.factor >= 1.0) || !std::isfinite(c.factor)))
        return fail(DRKV_ERR_INVALID, "rope_create: factor must be at least 1");
    if (c.scaling == DRKV_ROPE_BASE && c.rotary_dim < 4)
        return fail(DRKV_ERR_INVALID, "rope_create: base scaling needs a rotary_dim of at least 4");
    if ((c.scaling == DRKV_ROPE_BANDS || c.scaling == DRKV_ROPE_RAMP) && c.original_context < 1)
        return fail(DRKV_ERR_INVALID, "rope_create: original_context must be positive");
    if (c.scaling == DRKV_ROPE_BANDS && !(c.low_freq_factor > 0.f && c.high_freq_factor > c.low_freq_factor && std::isfinite(c.high_freq_factor)))
        return fail(DRKV_ERR_INVALID, "rope_create: bands need 0 < low_freq_factor < high_freq_factor");
    if (c.scaling == DRKV_ROPE_RAMP && !(c.beta_slow > 0.f && c.beta_fast > c.beta_slow && std::isfinite(c.beta_fast)))
        return fail(DRKV_ERR_INVALID, "rope_create: the ramp needs 0 < beta_slow < beta_fast");
    if (!(c.attention_factor >= 0.f) || !std::isfinite(c.attention_factor))
        return fail(DRKV_ERR_INVALID, "rope_create: attention_factor must be 0 (automatic) or positive");
    drkv_rope* r = new (std::nothrow) drkv_rope();
    if (!r) return fail(DRKV_ERR_CAPACITY, "rope_create: out of host memory");
    r->cfg = c;
    r->factor = c.attention_factor > 0.f ? c.attention_factor
                : c.scaling == DRKV_ROPE_RAMP ? (float)(0.1 * log(c.factor) + 1.0)
                                              : 1.f;
    std::vector<uint64_t> turns;
    try {
        std::vector<long double> f;
        frequencies(c, &f);
        turns.resize(f.size());
        for (size_t i = 0; i < f.size(); i++) {
            r->freq.push_back((double)f[i]);
            const long double t = f[i] / (2 * 3.141592653589793238462643383279502884L);
            const long double frac = t - floorl(t);
            turns[i] = frac >= 1.0L ? 0 : (uint64_t)ldexpl(frac, 64);
        }
    } catch (const std::bad_alloc&) {
        delete r;
        return fail(DRKV_ERR_CAPACITY, "rope_create: out of host memory");
    }
    if (c.device >= 0) {
        DeviceGuard dev(c.device);
        if (!dev.ok()) {
            delete r;
            return fail(DRKV_ERR_NO_DEVICE, "rope_create: cudaSetDevice failed");
        }
        if (cudaDeviceGetAttribute(&r->num_sms, cudaDevAttrMultiProcessorCount, c.device) != cudaSuccess ||
            cudaMalloc(&r->d_turns, turns.size() * 8) != cudaSuccess ||
            cudaMemcpy(r->d_turns, turns.data(), turns.size() * 8, cudaMemcpyHostToDevice) != cudaSuccess) {
            cudaFree(r->d_turns);
            cudaGetLastError();          // reported here
            delete r;
            return fail(DRKV_ERR_CUDA, "rope_create: allocating the frequency table failed");
        }
    }
    *out = r;
    return DRKV_OK;
}

void drkv_rope_destroy(drkv_rope* r) {
    if (!r) return;
    if (r->d_turns) {
        DeviceGuard dev(r->cfg.device);
        cudaDeviceSynchronize();
        cudaFree(r->d_turns);
    }
    delete r;
}

int drkv_rope_frequencies(const drkv_rope* r, double* out, int cap) {
    if (!r || cap < 0 || (cap > 0 && !out)) return fail(DRKV_ERR_INVALID, "rope_frequencies: bad argument");
    const int n = (int)r->freq.size() < cap ? (int)r->freq.size() : cap;
    for (int i = 0; i < n; i++) out[i] = r->freq[i];
    return (int)r->freq.size();
}

int drkv_rope_apply(const drkv_rope* r, int n_tokens, const int32_t* d_pos, const drkv_rope_rows* q, const drkv_rope_rows* k,
                    int inverse, void* stream) {
    if (!r || n_tokens < 0 || (!q && !k)) return fail(DRKV_ERR_INVALID, "rope_apply: bad argument");
    if (!r->d_turns) return fail(DRKV_ERR_NO_DEVICE, "rope_apply: the rotation was created without a device");
    const int d = r->cfg.head_dim, rot = r->cfg.rotary_dim;
    int vw = 8;
    while (vw > 1 && (rot / 2) % vw != 0) vw >>= 1;
    bool copies = false, wide_rows = true;                       // wide_rows: every row in 16-byte vectors
    for (const drkv_rope_rows* x : {q, k}) {
        if (!x || x->heads == 0) continue;
        if (x->heads < 0 || x->heads > 4096) return fail(DRKV_ERR_INVALID, "rope_apply: heads must be 0 to 4096");
        if (n_tokens == 0) continue;
        if (!x->src || !x->dst || reinterpret_cast<uintptr_t>(x->src) % 2 || reinterpret_cast<uintptr_t>(x->dst) % 2)
            return fail(DRKV_ERR_INVALID, "rope_apply: null or odd row pointer");
        if (x->src_token_stride < 0 || x->src_head_stride < 0)
            return fail(DRKV_ERR_INVALID, "rope_apply: negative stride");
        if (!rows_apart(x->dst_token_stride, x->dst_head_stride, n_tokens, x->heads, d))
            return fail(DRKV_ERR_INVALID, "rope_apply: rows of the destination overlap");
        const bool same = (n_tokens < 2 || x->src_token_stride == x->dst_token_stride) &&
                          (x->heads < 2 || x->src_head_stride == x->dst_head_stride);
        if (x->src != x->dst || !same) {
            // in place needs the very same rows; a source that merely overlaps the destination is refused
            auto last = [&](int64_t ts, int64_t hs) { return 2 * ((n_tokens - 1) * ts + (x->heads - 1) * hs + d); };
            const char *s0 = (const char*)x->src, *d0 = (const char*)x->dst;
            const char *s1 = s0 + last(x->src_token_stride, x->src_head_stride), *d1 = d0 + last(x->dst_token_stride, x->dst_head_stride);
            if (x->src == x->dst) return fail(DRKV_ERR_INVALID, "rope_apply: in place with different strides");
            // interleaved rows of one buffer (q and k of a fused projection written back beside them) may share a span
            // only when both step alike and never meet
            if (s0 < d1 && d0 < s1) {
                const int64_t gap = (d0 > s0 ? d0 - s0 : s0 - d0) / 2;
                const int64_t span = (int64_t)(x->heads - 1) * x->dst_head_stride + d;
                if (!(same && x->dst_head_stride <= x->dst_token_stride && gap >= span && gap + span <= x->dst_token_stride))
                    return fail(DRKV_ERR_INVALID, "rope_apply: source and destination overlap");
            }
            copies = true;
        }
        vw = widest(*x, n_tokens, vw);
        wide_rows &= widest(*x, n_tokens, 8) == 8;
    }
    const int qh = q ? q->heads : 0, kh = k ? k->heads : 0;
    if (n_tokens == 0 || qh + kh == 0) return DRKV_OK;
    if (!d_pos || reinterpret_cast<uintptr_t>(d_pos) % 4) return fail(DRKV_ERR_INVALID, "rope_apply: null or unaligned positions");
    RopeParams p{};
    auto rows = [](const drkv_rope_rows& x) {
        return RopeRowsDev{x.src, x.dst, x.src_token_stride, x.src_head_stride, x.dst_token_stride, x.dst_head_stride};
    };
    if (q) p.q = rows(*q);
    if (k) p.k = rows(*k);
    p.pos = d_pos;
    p.turns = r->d_turns;
    p.n_tokens = n_tokens;
    p.q_heads = qh;
    p.heads = qh + kh;
    p.half = rot / 2;
    p.rotary_dim = rot;
    p.pairs_layout = r->cfg.layout == DRKV_ROPE_PAIRS;
    p.inverse = inverse != 0;
    p.factor = r->factor;
    p.rot_items = p.half / vw;
    p.row_items = p.rot_items + (copies ? (d - rot) / vw : 0);   // head_dim is a multiple of 8, rotary_dim of 2 vw
    p.magic_row = magic_of(p.row_items);
    // Several tokens share a CTA once one each would be more than two waves of CTAs (8 of 256 threads an SM).
    p.tokens_per_cta = 1;
    while (p.tokens_per_cta < 8 && (int64_t)n_tokens > (int64_t)r->num_sms * 16 * p.tokens_per_cta) p.tokens_per_cta *= 2;
    while (p.tokens_per_cta > 1 && (int64_t)p.tokens_per_cta * p.heads * p.row_items > (1 << 16)) p.tokens_per_cta /= 2;
    // the row kernel takes heads of 64, 128 and 256 dims (their lanes divide a warp) in 16-byte vectors
    const bool by_rows = wide_rows && (d == 64 || d == 128 || d == 256);
    const int mode = p.pairs_layout ? kPairs : rot % 16 == 0 ? kHalves : kAnyHalves;
    const int ctas = (n_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
    // Few tokens: the heads are spread over CTAs too, as many as go at once in each (one token of 72 heads of 128: 1.8 us, in one CTA 3.3).
    const int at_once = by_rows ? kRopeThreads / (d / 8) : p.row_items < kRopeThreads ? kRopeThreads / p.row_items : 1;
    int parts = (p.heads + at_once - 1) / at_once;
    if (parts > 2 * r->num_sms / ctas) parts = 2 * r->num_sms / ctas > 0 ? 2 * r->num_sms / ctas : 1;
    p.heads_per_cta = (p.heads + parts - 1) / parts;
    p.magic_heads = magic_of(p.heads_per_cta);
    const dim3 grid(ctas, (p.heads + p.heads_per_cta - 1) / p.heads_per_cta);
    const int pad = by_rows && mode == kAnyHalves ? (rot + 7) & ~7 : (p.half + 3) & ~3;
    size_t smem = (size_t)p.tokens_per_cta * 2 * pad * sizeof(float);
    DeviceGuard dev(r->cfg.device);
    if (!dev.ok()) return fail(DRKV_ERR_CUDA, "rope_apply: cudaSetDevice failed");
    if (by_rows) {
        const int lg = d == 64 ? 3 : d == 128 ? 4 : 5;
        if (mode == kAnyHalves) smem += (size_t)(kRopeThreads >> lg) * ring_elements(1 << lg) * 2;
        const cudaStream_t st = (cudaStream_t)stream;
        const cudaError_t e = r->cfg.dtype == DRKV_DTYPE_F16 ? launch_rows<__half>(p, mode, lg, grid, smem, st)
                                                             : launch_rows<__nv_bfloat16>(p, mode, lg, grid, smem, st);
        if (e != cudaSuccess) return fail(DRKV_ERR_CUDA, cudaGetErrorString(e));
        return DRKV_OK;
    }
    const cudaError_t ce = r->cfg.dtype == DRKV_DTYPE_F16 ? launch_rope<__half>(p, vw, grid, smem, (cudaStream_t)stream)
                                                          : launch_rope<__nv_bfloat16>(p, vw, grid, smem, (cudaStream_t)stream);
    if (ce != cudaSuccess) return fail(DRKV_ERR_CUDA, cudaGetErrorString(ce));
    return DRKV_OK;
}

}  // extern "C"
