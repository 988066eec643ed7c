// rope_append.cu - the rotary step of a step's q and k rows, with the heads' RMS norms before it, and the append of its k and v rows to
// the paged cache, one launch.
//
// A head row of D values is D / 2 couples; a lane has W neighbouring ones (8 of bf16 rows, 4 of fp32 rows or where the pairs or starts do
// not come in eights), in two vectors of W values: i .. and i + rot / 2 .. where pairs lie half a turn's width apart, 2i .. 2i + 2W - 1
// where they are neighbours and where values pass unturned.  So D / (2W) lanes have a row, its norm is a butterfly among them, and every load
// and store is a vector.  The angle's sine and cosine belong to (token, pair) and serve all heads: a block makes them once for its tokens,
// while its first rows are under way, and asks for a row's successor before it turns the row.  pos * inv_freq is taken in 64 bits and
// reduced to one turn there: a product in fp32 is off by 4e-3 radians at position 131072 already.
//
// Long calls are bound by HBM and, before it, by the wait for a row's loads (half of the issue slots are used) and the instructions around two
// vectors a lane; short ones by latency.  On a B200: 4096 tokens, 32 / 8 heads of 128, bf16, pairs as neighbours on three axes, 101 MB:
// 22 us, 4.6 TB/s (four values a lane 29); 64 tokens of fp32 rows with norms into e4m3: 2.9 us (one block a token 6.0); one token 2.3 us.
#include "paged.cuh"
#include "pdl.cuh"

#include <cuda_fp8.h>

namespace bsx {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 16;  // most tokens a block takes
constexpr int kRopeBlocks = 4;   // an SM

struct RopeParams {
    const void *q, *k, *v;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
    const int64_t* slot;
    const int32_t* pos;
    int64_t pos_stride;
    const float* inv_freq;
    const int32_t* pair_axis;
    const float *q_norm, *k_norm, *k_scale, *v_scale;
    void* q_out;
    void *k_cache, *v_cache;
    int64_t k_page, v_page, n_slots;
    int32_t* status;
    float magnitude, eps;
    int32_t T, hq, hk, rot, n_axes, interleaved, page_shift, tokens;   // tokens: a block's
};

template <int W, bool BF16, bool VEC>
__device__ __forceinline__ void load_values(const void* base, int64_t at, float (&x)[W]) {
    if constexpr (BF16) {
        const uint16_t* s = static_cast<const uint16_t*>(base) + at;
        if constexpr (VEC) {
            uint32_t w[W / 2];
            if constexpr (W == 8) {
                const uint4 u = *reinterpret_cast<const uint4*>(s);
                w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(s);
                w[0] = u.x, w[1] = u.y;
            }
#pragma unroll
            for (int i = 0; i < W / 2; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) x[i] = __uint_as_float((uint32_t) s[i] << 16);
        }
    } else {
        const float* s = static_cast<const float*>(base) + at;
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            if constexpr (VEC) {
                const float4 u = *reinterpret_cast<const float4*>(s + i);
                x[i] = u.x, x[i + 1] = u.y, x[i + 2] = u.z, x[i + 3] = u.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i + j] = s[i + j];
            }
        }
    }
}

template <int W>
__device__ __forceinline__ void store_bf16(uint16_t* to, const float (&x)[W]) {
    uint32_t w[W / 2];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (W == 8) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
}
// the quotient, not a product with a reciprocal: a value halfway between two codes goes where the definition sends it
template <int W>
__device__ __forceinline__ void store_e4m3(uint8_t* to, const float (&x)[W], float scale) {
    uint32_t w[W / 4];
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] / scale, x[4 * i + 1] / scale), __NV_SATFINITE, __NV_E4M3);
        const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] / scale, x[4 * i + 3] / scale), __NV_SATFINITE, __NV_E4M3);
        w[i] = a | b << 16;
    }
    if constexpr (W == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(to) = w[0];
}

constexpr int lanes_of(int d, int w) { return d / (2 * w) <= 4 ? 4 : d / (2 * w) <= 8 ? 8 : d / (2 * w) <= 16 ? 16 : 32; }   // of a row; 192 values leave a quarter idle

template <int D, int W, bool BF16, bool VEC, bool E4M3>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const RopeParams p) {
    constexpr int kLanes = lanes_of(D, W), kRows = kRopeThreads / kLanes;
    __shared__ float2 turn[kRopeTokens][D / 2];
    pdl_wait();
    const int half = p.rot >> 1;
    const int t0 = blockIdx.x * p.tokens, nt = min(p.tokens, p.T - t0);
    const int part = threadIdx.x & (kLanes - 1);
    const bool works = part < D / (2 * W);
    const int c = works ? part * W : 0;   // the lane's first couple
    const bool turns = c < half;
    const bool apart = turns && !p.interleaved;
    const int o1 = apart ? c : 2 * c, o2 = apart ? c + half : 2 * c + W;
    const int heads = p.hq + 2 * p.hk, step = gridDim.y * kRows;
    // a lane's share of a row: q's, then k's, then v's heads of a token
    struct Row {
        int t, h;   // token of the block, head
    };
    auto further = [&](Row r, int n) {
        r.h += n;
        while (r.h >= heads) r.h -= heads, ++r.t;
        return r;
    };
    auto load = [&](const Row& r, float (&a)[W], float (&b)[W]) {
        const int64_t token = t0 + r.t;
        const bool q = r.h < p.hq, v = r.h >= p.hq + p.hk;
        const void* src = q ? p.q : v ? p.v : p.k;
        const int head = q ? r.h : v ? r.h - p.hq - p.hk : r.h - p.hq;
        const int64_t at = token * (q ? p.q_tok : v ? p.v_tok : p.k_tok) + (int64_t) head * (q ? p.q_head : v ? p.v_head : p.k_head);
        load_values<W, BF16, VEC>(src, at + (v ? 2 * c : o1), a);
        load_values<W, BF16, VEC>(src, at + (v ? 2 * c + W : o2), b);
    };
    auto finish = [&](const Row& r, bool there, float (&a)[W], float (&b)[W]) {
        const bool q = r.h < p.hq, v = r.h >= p.hq + p.hk;
        if (p.q_norm || p.k_norm) {
            const float* w = q ? p.q_norm : v ? nullptr : p.k_norm;
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) sq += a[i] * a[i] + b[i] * b[i];
#pragma unroll
            for (int m = kLanes / 2; m; m >>= 1) sq += __shfl_xor_sync(kFull, sq, m);
            if (w) {
                const float f = rsqrtf(sq / D + p.eps);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    a[i] *= f * w[o1 + i];
                    b[i] *= f * w[o2 + i];
                }
            }
        }
        if (!there) return;
        if (!v && turns) {
            const float2* cs = &turn[r.t][c];
            if (apart) {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const float2 e = cs[i];
                    const float u = a[i] * e.x - b[i] * e.y;
                    b[i] = a[i] * e.y + b[i] * e.x;
                    a[i] = u;
                }
            } else {
#pragma unroll
                for (int i = 0; i < W; i += 2) {
                    const float2 e = cs[i / 2], f = cs[i / 2 + W / 2];
                    const float u = a[i] * e.x - a[i + 1] * e.y, g = b[i] * f.x - b[i + 1] * f.y;
                    a[i + 1] = a[i] * e.y + a[i + 1] * e.x;
                    b[i + 1] = b[i] * f.y + b[i + 1] * f.x;
                    a[i] = u;
                    b[i] = g;
                }
            }
        }
        const int64_t token = t0 + r.t;
        if (q) {
            uint16_t* out = static_cast<uint16_t*>(p.q_out) + (token * p.hq + r.h) * D;
            store_bf16<W>(out + o1, a);
            store_bf16<W>(out + o2, b);
            return;
        }
        const int64_t slot = p.slot[token];
        if (slot < 0 || slot >= p.n_slots) {
            if (slot >= 0 && p.status && part == 0) atomicOr(p.status, BSX_PAGED_BAD_SLOT);
            return;
        }
        const int head = r.h - p.hq - (v ? p.hk : 0), place = (int) slot & ((1 << p.page_shift) - 1);
        const int64_t at = (slot >> p.page_shift) * (v ? p.v_page : p.k_page) + ((head << p.page_shift) + place) * D;
        void* cache = v ? p.v_cache : p.k_cache;
        const int p1 = v ? 2 * c : o1, p2 = v ? 2 * c + W : o2;
        if (E4M3) {
            const float scale = (v ? p.v_scale : p.k_scale)[head];
            uint8_t* out = static_cast<uint8_t*>(cache) + at;
            store_e4m3<W>(out + p1, a, scale);
            store_e4m3<W>(out + p2, b, scale);
        } else {
            uint16_t* out = static_cast<uint16_t*>(cache) + at;
            store_bf16<W>(out + p1, a);
            store_bf16<W>(out + p2, b);
        }
    };
    Row now = further(Row{0, 0}, blockIdx.y * kRows + threadIdx.x / kLanes);
    float a[W], b[W];
#pragma unroll
    for (int i = 0; i < W; ++i) a[i] = b[i] = 0.f;
    if (works && now.t < nt) load(now, a, b);   // under way while the angles are made
    for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
        const int t = i / half, pair = i - t * half;
        const int axis = p.pair_axis ? min(max(p.pair_axis[pair], 0), p.n_axes - 1) : 0;
        const double turned = (double) p.pos[axis * p.pos_stride + t0 + t] * (double) p.inv_freq[pair] * 0.15915494309189533577;
        float s, co;
        sincospif((float) (2.0 * (turned - rint(turned))), &s, &co);
        turn[t][pair] = make_float2(co * p.magnitude, s * p.magnitude);
    }
    __syncthreads();
    // rows of a warp go round together: the butterfly needs its lanes
    for (int first = blockIdx.y * kRows; first < nt * heads; first += step) {
        const Row next = further(now, step);
        float a2[W], b2[W];
#pragma unroll
        for (int i = 0; i < W; ++i) a2[i] = b2[i] = 0.f;
        if (works && next.t < nt) load(next, a2, b2);
        finish(now, works && now.t < nt, a, b);
        now = next;
#pragma unroll
        for (int i = 0; i < W; ++i) a[i] = a2[i], b[i] = b2[i];
    }
}

template <int D, int W, bool BF16, bool VEC>
void launch_rope(const RopeParams& p, bool e4m3, dim3 grid, cudaStream_t st) {
    if (e4m3) launch_early(rope_append_kernel<D, W, BF16, VEC, true>, grid, dim3(kRopeThreads), 0, st, p);
    else launch_early(rope_append_kernel<D, W, BF16, VEC, false>, grid, dim3(kRopeThreads), 0, st, p);
}
template <int D>
void launch_rope(const RopeParams& p, bool bf16, bool wide, bool vec, bool e4m3, dim3 grid, cudaStream_t st) {
    if (bf16 && wide) launch_rope<D, 8, true, true>(p, e4m3, grid, st);
    else if (bf16) vec ? launch_rope<D, 4, true, true>(p, e4m3, grid, st) : launch_rope<D, 4, true, false>(p, e4m3, grid, st);
    else vec ? launch_rope<D, 4, false, true>(p, e4m3, grid, st) : launch_rope<D, 4, false, false>(p, e4m3, grid, st);
}

}  // namespace
}  // namespace bsx

using namespace bsx;

extern "C" int32_t bsx_rope_append(const bsx_kv_cache* cache, const bsx_rope* rope, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                   int32_t n_q_heads, const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                   int64_t v_token_stride, int64_t v_head_stride, int32_t x_kind, int32_t T, const int64_t* slot, const int32_t* pos,
                                   int64_t pos_stride, int32_t n_axes, const float* q_norm, const float* k_norm, float eps, void* q_out,
                                   int32_t* status, void* stream) {
    if (!stream) return BSX_E_STREAM;
    if (x_kind != BSX_X_F32 && x_kind != BSX_X_BF16) return BSX_E_TYPE;
    const int32_t bad = cache_status(cache);
    if (bad) return bad;
    if (!rope) return BSX_E_POINTER;
    const int D = cache->head_dim;
    const bool append = k || v;
    if (rope->rot_dim < 0 || rope->rot_dim > D || rope->rot_dim % 8 || n_q_heads < 0 || T < 0) return BSX_E_GEOMETRY;
    if (rope->rot_dim && (n_axes < 1 || n_axes > 4)) return BSX_E_GEOMETRY;
    if (n_q_heads > 1024 || T > BSX_PAGED_MAX_TOKENS) return BSX_E_LIMIT;
    if (T == 0 || (n_q_heads == 0 && !append)) return BSX_OK;
    if (rope->rot_dim && (!rope->inv_freq || !pos)) return BSX_E_POINTER;
    if (n_q_heads && (!q || !aligned(q_out, 16))) return BSX_E_POINTER;
    if (append && (!k || !v || !slot)) return BSX_E_POINTER;
    const size_t elem = x_kind == BSX_X_BF16 ? 2 : 4;
    if ((n_q_heads && !aligned(q, elem)) || (append && (!aligned(k, elem) || !aligned(v, elem)))) return BSX_E_POINTER;
    RopeParams p{};
    p.q = q, p.k = k, p.v = v;
    p.q_tok = q_token_stride, p.q_head = q_head_stride, p.k_tok = k_token_stride, p.k_head = k_head_stride;
    p.v_tok = v_token_stride, p.v_head = v_head_stride;
    p.slot = slot, p.pos = pos, p.pos_stride = pos_stride;
    p.inv_freq = rope->inv_freq, p.pair_axis = rope->pair_axis, p.q_norm = q_norm, p.k_norm = k_norm;
    p.k_scale = cache->k_scale, p.v_scale = cache->v_scale;
    p.q_out = q_out, p.k_cache = cache->k, p.v_cache = cache->v;
    p.k_page = cache->k_page_stride, p.v_page = cache->v_page_stride, p.n_slots = cache->n_pages * cache->page_size;
    p.status = status, p.magnitude = rope->magnitude, p.eps = eps;
    p.T = T, p.hq = n_q_heads, p.hk = append ? cache->n_kv_heads : 0, p.rot = rope->rot_dim, p.n_axes = n_axes;
    p.interleaved = rope->interleaved;
    p.page_shift = log2_of(cache->page_size);
    // vectors where every row's start allows them, of 16 bytes where the pairs of bf16 rows come in eights
    const bool bf16 = x_kind == BSX_X_BF16, e4m3 = cache->kind == BSX_KV_E4M3;
    auto starts = [&](int n) {
        bool ok = true;
        if (n_q_heads) ok = ok && aligned(q, n * elem) && q_token_stride % n == 0 && q_head_stride % n == 0;
        if (append)
            ok = ok && aligned(k, n * elem) && aligned(v, n * elem) && k_token_stride % n == 0 && k_head_stride % n == 0 && v_token_stride % n == 0 &&
                 v_head_stride % n == 0;
        return ok;
    };
    const bool vec = starts(4), wide = bf16 && rope->rot_dim % 16 == 0 && starts(8);
    // A block takes as many tokens as make one wave of four blocks an SM (their registers let no more on; 4096 tokens of 48 rows: 22 us, for
    // three blocks an SM 25, for five 29), and enough to have rows for all of its threads; while there are fewer blocks than that, the rounds
    // of a block's rows are shared out (64 tokens of 80 rows: 3.0 us, a block a token 6.0)
    const int rows = kRopeThreads / lanes_of(D, wide ? 8 : 4), heads = n_q_heads + 2 * p.hk, full = (rows + heads - 1) / heads;
    const int even = (T + kRopeBlocks * 148 - 1) / (kRopeBlocks * 148);
    p.tokens = even > full ? even : full;
    if (p.tokens > kRopeTokens) p.tokens = kRopeTokens;
    const int blocks = (T + p.tokens - 1) / p.tokens, rounds = (p.tokens * heads + rows - 1) / rows;
    int share = blocks < kRopeBlocks * 148 ? kRopeBlocks * 148 / blocks : 1;
    if (share > rounds) share = rounds;
    const dim3 grid((unsigned) blocks, (unsigned) share);
    cudaStream_t st = (cudaStream_t) stream;
    switch (D) {
        case 64: launch_rope<64>(p, bf16, wide, vec, e4m3, grid, st); break;
        case 128: launch_rope<128>(p, bf16, wide, vec, e4m3, grid, st); break;
        case 192: launch_rope<192>(p, bf16, wide, vec, e4m3, grid, st); break;
        default: launch_rope<256>(p, bf16, wide, vec, e4m3, grid, st); break;
    }
    return launch_status();
}
