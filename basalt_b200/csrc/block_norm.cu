// block_norm.cu - the norms around an attention or expert block: of the block's output row y and the residual row x,
//   z = y / rms(y) * post_w,   h = residual_scale * x + block_scale * gate * z,   xn = h / rms(h) * pre_w.
//
// Bound by HBM: y, x (and a gate per token) in, h and xn out, each once.  A row is one block's, its values stay in registers from the first
// load to the last store: y, x and gate are requested together, the first sum goes round while the others are still under way.  A thread
// takes vectors of four values, up to kVectors of them, the block's threads side by side; where a row's start or length is no multiple of
// four it reads and writes the same four one by one.  Sums: a thread's values, a warp's threads by butterfly, the warps in a fixed order: the
// same for every T, stride and start.
//
// On a B200: 8192 rows of 7168, y bf16, x fp32, a gate for all, bf16 rows out, 705 MB: 121 us, 5.8 TB/s; 16384 of 7168, all fp32: 311 us,
// 6.8 TB/s; one row of 2048 3.0 us; rows of 4097 bf16 values, one by one, 93 us for 4096 (30 at the rate of the others).  Rows staged
// in shared memory by asynchronous copies, a block going from row to row: 164 us where this takes 121.
#include "common.cuh"
#include "pdl.cuh"

#include <type_traits>

#include <cuda_bf16.h>

namespace bsx {
namespace {

struct BlockNormParams {
    const void *y, *x, *gate;
    const float *post_w, *pre_w;
    void *h, *act;
    float* xn;
    int64_t y_stride, x_stride, gate_stride, h_stride;   // bytes
    float eps, block_scale, residual_scale, inv_k;
    int32_t K, gate_sigmoid;
};

// Four values of a row as they lie in memory: vector v of it, of which the columns below K are there; in one access where VEC, else one each
template <bool BF16, bool VEC>
struct Four {
    uint32_t w[BF16 ? 2 : 4];
    __device__ __forceinline__ void load(const char* row, uint32_t v, int K) {
        const char* s = row + v * (BF16 ? 8u : 16u);
        if constexpr (!VEC) {
            zero();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if ((int) v * 4 + j >= K) continue;
                if constexpr (BF16) w[j / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(s)[j] << (j % 2 * 16);
                else w[j] = reinterpret_cast<const uint32_t*>(s)[j];
            }
        } else if constexpr (BF16) {
            const uint2 u = *reinterpret_cast<const uint2*>(s);
            w[0] = u.x, w[1] = u.y;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(s);
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < (BF16 ? 2 : 4); ++j) w[j] = 0;
    }
    __device__ __forceinline__ float operator[](int j) const {
        if constexpr (BF16) return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        else return __uint_as_float(w[j]);
    }
};
template <bool BF16, bool VEC>
__device__ __forceinline__ void store4(char* row, uint32_t v, int K, const float (&x)[4]) {
    char* s = row + v * (BF16 ? 8u : 16u);
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if ((int) v * 4 + j >= K) continue;
            if (BF16) reinterpret_cast<__nv_bfloat16*>(s)[j] = __float2bfloat16_rn(x[j]);
            else reinterpret_cast<float*>(s)[j] = x[j];
        }
    } else if constexpr (BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        *reinterpret_cast<uint2*>(s) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        *reinterpret_cast<float4*>(s) = make_float4(x[0], x[1], x[2], x[3]);
    }
}

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum_xor(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < (int) blockDim.x / 32; i += 4) {   // past the last warp zeros stand
        const float4 v = *reinterpret_cast<const float4*>(red + i);
        s = ((s + v.x) + v.y) + (v.z + v.w);
    }
    return s;
}

template <bool VEC, int kVectors, bool Y16, bool X16, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) block_norm_kernel(const BlockNormParams p) {
    __shared__ __align__(16) float red[2][32];
    pdl_wait();
    const int64_t t = blockIdx.x;
    const uint32_t threads = blockDim.x, n = (uint32_t) (p.K + 3) / 4;
    const char* const y_row = static_cast<const char*>(p.y) + t * p.y_stride;
    const char* const x_row = static_cast<const char*>(p.x) + t * p.x_stride;
    const char* const gate_row = static_cast<const char*>(p.gate) + t * p.gate_stride;
    Four<Y16, VEC> y[kVectors];
    Four<X16, VEC> x[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const uint32_t v = threadIdx.x + i * threads;
        y[i].zero();
        if (v < n) y[i].load(y_row, v, p.K);
    }
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const uint32_t v = threadIdx.x + i * threads;
        x[i].zero();
        if (p.x && v < n) x[i].load(x_row, v, p.K);
    }
    constexpr bool kGateEarly = kVectors <= 2 || Y16;   // where the registers suffice
    Four<Y16, VEC> gate[kGateEarly ? kVectors : 1];
    if (kGateEarly && p.gate) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const uint32_t v = threadIdx.x + i * threads;
            if (v < n) gate[kGateEarly ? i : 0].load(gate_row, v, p.K);
        }
    }
    if (threadIdx.x < 64 && (threadIdx.x & 31) >= threads / 32) red[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
    if (threads == 32 && threadIdx.x) red[1][threadIdx.x] = 0.f;
    float scale = p.block_scale;
    if (p.post_w) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sq = fmaf(y[i][j], y[i][j], sq);
        scale *= rsqrtf(block_sum(sq, red[0]) * p.inv_k + p.eps);
    }
    float h[kVectors][4], sq = 0.f;
    char* const h_row = static_cast<char*>(p.h) + t * p.h_stride;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const uint32_t v = threadIdx.x + i * threads;
        if (v >= n) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) h[i][j] = y[i][j] * scale;
        if (p.post_w) {
            Four<false, VEC> w;
            w.load(reinterpret_cast<const char*>(p.post_w), v, p.K);
#pragma unroll
            for (int j = 0; j < 4; ++j) h[i][j] *= w[j];
        }
        if (p.gate) {
            Four<Y16, VEC> g = gate[kGateEarly ? i : 0];
            if (!kGateEarly) g.load(gate_row, v, p.K);
            if (p.gate_sigmoid) {
#pragma unroll
                for (int j = 0; j < 4; ++j) h[i][j] *= __fdividef(1.f, 1.f + expf(-g[j]));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) h[i][j] *= g[j];
            }
        }
        if (p.x) {
#pragma unroll
            for (int j = 0; j < 4; ++j) h[i][j] = fmaf(p.residual_scale, x[i][j], h[i][j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sq = fmaf(h[i][j], h[i][j], sq);
        store4<X16, VEC>(h_row, v, p.K, h[i]);
    }
    if (!p.pre_w) return;
    const float s = rsqrtf(block_sum(sq, red[1]) * p.inv_k + p.eps);
    char* const xn_row = reinterpret_cast<char*>(p.xn) + t * p.K * 4;
    char* const act_row = static_cast<char*>(p.act) + t * p.K * 2;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const uint32_t v = threadIdx.x + i * threads;
        if (v >= n) continue;
        Four<false, VEC> w;
        w.load(reinterpret_cast<const char*>(p.pre_w), v, p.K);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[i][j] *= s * w[j];
        if (p.xn) store4<false, VEC>(xn_row, v, p.K, h[i]);
        if (p.act) store4<true, VEC>(act_row, v, p.K, h[i]);
    }
}

template <bool VEC, int kVectors, int kThreads>
void launch_norm(const BlockNormParams& p, bool y16, bool x16, int T, int threads, cudaStream_t st) {
    if (y16) {
        if (x16) launch_early(block_norm_kernel<VEC, kVectors, true, true, kThreads>, dim3(T), dim3(threads), 0, st, p);
        else launch_early(block_norm_kernel<VEC, kVectors, true, false, kThreads>, dim3(T), dim3(threads), 0, st, p);
    } else {
        if (x16) launch_early(block_norm_kernel<VEC, kVectors, false, true, kThreads>, dim3(T), dim3(threads), 0, st, p);
        else launch_early(block_norm_kernel<VEC, kVectors, false, false, kThreads>, dim3(T), dim3(threads), 0, st, p);
    }
}

}  // namespace
}  // namespace bsx

using namespace bsx;

extern "C" int32_t bsx_block_norm(const void* y, int32_t y_kind, int64_t y_stride, const void* x, int32_t x_kind, int64_t x_stride, const void* gate,
                                  int64_t gate_stride, int32_t gate_sigmoid, const float* post_w, const float* pre_w, float eps, float block_scale,
                                  float residual_scale, int64_t K, int32_t T, void* h, int64_t h_stride, void* act, float* xn, void* stream) {
    if (!stream) return BSX_E_STREAM;
    if ((y_kind != BSX_X_F32 && y_kind != BSX_X_BF16) || (x_kind != BSX_X_F32 && x_kind != BSX_X_BF16)) return BSX_E_TYPE;
    if (K <= 0 || T < 0 || y_stride < 0 || (x && x_stride < 0) || gate_stride < 0 || (T > 1 && h_stride < K)) return BSX_E_GEOMETRY;
    if (K > 16384) return BSX_E_LIMIT;
    if (T == 0) return BSX_OK;
    const bool y16 = y_kind == BSX_X_BF16, x16 = x_kind == BSX_X_BF16;
    const size_t ey = y16 ? 2 : 4, ex = x16 ? 2 : 4;
    if (!aligned(y, ey) || (x && !aligned(x, ex)) || (gate && !aligned(gate, ey)) || !aligned(h, ex) || (post_w && !aligned(post_w, 4)) ||
        (pre_w && !aligned(pre_w, 4)) || (act && !aligned(act, 2)) || (xn && !aligned(xn, 4)))
        return BSX_E_POINTER;
    if (pre_w ? !act && !xn : act || xn) return BSX_E_POINTER;
    const int64_t by = (int64_t) ey, bx = (int64_t) ex;
    const BlockNormParams p{y,  x,   gate,        post_w,         pre_w,            h, act, xn, y_stride * by, x_stride * bx, gate_stride * by, h_stride * bx,
                            eps, block_scale, residual_scale, 1.f / (float) K, (int32_t) K, gate_sigmoid};
    auto by4 = [](const void* a, size_t e, int64_t stride) { return !a || (aligned(a, 4 * e) && stride % 4 == 0); };
    const bool vec = K % 4 == 0 && by4(y, ey, y_stride) && by4(x, ex, x_stride) && by4(gate, ey, gate_stride) && by4(h, ex, h_stride) && by4(post_w, 4, 0) &&
                     by4(pre_w, 4, 0) && by4(act, 2, 0) && by4(xn, 4, 0);
    cudaStream_t st = (cudaStream_t) stream;
    const int units = (int) ((K + 3) / 4);
    // vectors a thread: one, two, four, by the width alone, so that a row's sums do not depend on the call (us for 16384 rows, y bf16, with a
    // gate: 2048 wide one 91, two 71, four 66, but one row 2.9, 3.4, 4.5; 7168 wide two 388, four 271)
    const int each = units <= 256 ? 1 : units <= 512 ? 2 : 4;
    const int threads = ((units + each - 1) / each + 31) / 32 * 32;
    auto go = [&](auto v) {
        constexpr bool kVec = decltype(v)::value;
        if (each == 1) launch_norm<kVec, 1, 256>(p, y16, x16, T, threads, st);
        else if (each == 2) launch_norm<kVec, 2, 256>(p, y16, x16, T, threads, st);
        else if (threads <= 512) launch_norm<kVec, 4, 512>(p, y16, x16, T, threads, st);
        else launch_norm<kVec, 4, 1024>(p, y16, x16, T, threads, st);
    };
    if (vec) go(std::true_type{});
    else go(std::false_type{});
    return launch_status();
}
