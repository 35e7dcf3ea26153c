// Root-mean-square norm with the residual's addition, and rows brought to e4m3: h = x + skip, y = h / sqrt(mean(h^2) + eps) gamma, out as fp16 or as e4m3 codes
// with a scale for each 128 features of a row (the largest size of the 128 / 448, so that it becomes the largest code). Without the norm, y = x.
//
// One pass: a CTA has a row, a thread 8 features of it at a time (16 bytes), all in registers between the sum of squares and the codes. 16 neighbouring lanes
// have the 128 features of a scale, so its maximum takes four exchanges. Bound by memory: x and skip are read, residual (2 bytes) and codes (1 byte) written.
// Everything between is fp32; the norm is taken of the sum before it is rounded to fp16 for the residual.
#include "common.h"
#include "ptx.cuh"
#include "vec_math.cuh"

namespace et {
namespace {

constexpr int kScaleBlock = 128;       // features that share a scale
constexpr float kE4m3Max = 448.f;
constexpr int kMaxWidth = 32768;       // a row of the general kernel lies in shared memory

struct RowParams {
    void* out;
    const half *x, *skip, *gamma;
    half* residual;
    float* scales;                     // [blocks of 128][rows]
    long long out_pitch, x_pitch, skip_pitch, residual_pitch;
    int rows, width;
    float eps;
};

// The rounded quotient y / d, as what y * (about 1 / d) leaves of y is added to it, divided the same way.
__device__ __forceinline__ float quotient(float y, float d, float inverse) {
    const float q = y * inverse;
    return fmaf(fmaf(-q, d, y), inverse, q);
}
__device__ __forceinline__ float2 quotient2(float a, float b, float d, float inverse) {
    const float2 y = make_float2(a, b), i2 = make_float2(inverse, inverse), q = mul2(y, i2);
    return fma2(fma2(q, make_float2(-d, -d), y), i2, q);
}
// The scale of features whose largest size is `top` (/ 448), and about 1 / scale. Codes are those of rounded quotients y / scale, since fp16 features often lie in the middle between two codes:
// y * (448 / top) is one step beside it in some 70 of a million. A maximum that is infinite or not a number leaves a scale that is not a number.
struct Scale {
    float scale, inverse;
    __device__ __forceinline__ explicit Scale(float top) : scale(quotient(top, kE4m3Max, 1.f / kE4m3Max)) {
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
        if (top == 0.f) inverse = 0.f;
    }
};
__device__ __forceinline__ uint32_t e4m3_pair(float2 v) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(v.y), "f"(v.x));
    return d;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A row to a CTA, kV granules of 8 features to a thread; rows and pitches of whole granules.
template <int kV, bool kNorm, bool kSkip, bool kCodes>
__global__ void __launch_bounds__(kV == 4 ? 512 : 256) row_kernel(const __grid_constant__ RowParams p) {
    __shared__ float warp_sums[32];
    const int tid = threadIdx.x, lane = tid & 31, granules = p.width >> 3;
    const long long row = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    uint4 xv[kV], sv[kV], gv[kV];
#pragma unroll
    for (int v = 0; v < kV; ++v) {
        const int g = v * (int)blockDim.x + tid;
        if (g < granules) {
            xv[v] = *reinterpret_cast<const uint4*>(p.x + row * p.x_pitch + g * 8);
            if constexpr (kSkip) sv[v] = *reinterpret_cast<const uint4*>(p.skip + row * p.skip_pitch + g * 8);
        } else {
            xv[v] = sv[v] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    if constexpr (kNorm) {
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int g = v * (int)blockDim.x + tid;
            gv[v] = g < granules ? __ldg(reinterpret_cast<const uint4*>(p.gamma + g * 8)) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    float h[kV][8], sum = 0.f;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
        const half2 *const a = reinterpret_cast<const half2*>(&xv[v]), *const b = reinterpret_cast<const half2*>(&sv[v]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 y = __half22float2(a[i]);
            if constexpr (kSkip) {
                const float2 z = __half22float2(b[i]);
                y.x += z.x;
                y.y += z.y;
            }
            h[v][2 * i] = y.x;
            h[v][2 * i + 1] = y.y;
            sum = fmaf(y.x, y.x, sum);
            sum = fmaf(y.y, y.y, sum);
        }
    }
    float factor = 1.f;
    if constexpr (kNorm) {
        if (p.residual) {
#pragma unroll
            for (int v = 0; v < kV; ++v) {
                const int g = v * (int)blockDim.x + tid;
                uint4 r;
                half2* const o = reinterpret_cast<half2*>(&r);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = __floats2half2_rn(h[v][2 * i], h[v][2 * i + 1]);
                if (g < granules) *reinterpret_cast<uint4*>(p.residual + row * p.residual_pitch + g * 8) = r;
            }
        }
        sum = warp_sum(sum);
        const int warps = blockDim.x >> 5;
        if (warps > 1) {
            if (lane == 0) warp_sums[tid >> 5] = sum;
            __syncthreads();
            sum = warp_sum(lane < warps ? warp_sums[lane] : 0.f);
        }
        factor = rsqrtf(sum / (float)p.width + p.eps);
    }
#pragma unroll
    for (int v = 0; v < kV; ++v) {
        const int g = v * (int)blockDim.x + tid;
        if constexpr (kNorm) {
            const half2* const w = reinterpret_cast<const half2*>(&gv[v]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 s = __half22float2(w[i]);
                h[v][2 * i] = h[v][2 * i] * factor * s.x;
                h[v][2 * i + 1] = h[v][2 * i + 1] * factor * s.y;
            }
        }
        if constexpr (kCodes) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(h[v][i]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            const Scale s(top);
            if (g < granules) {
                uint2 c;
                auto two = [&](int i) { return e4m3_pair(quotient2(h[v][i], h[v][i + 1], s.scale, s.inverse)); };
                c.x = two(0) | two(2) << 16;
                c.y = two(4) | two(6) << 16;
                *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + row * p.out_pitch + g * 8) = c;
                if ((lane & 15) == 0) p.scales[(long long)(g >> 4) * p.rows + row] = s.scale;
            }
        } else if (g < granules) {
            uint4 r;
            half2* const o = reinterpret_cast<half2*>(&r);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __floats2half2_rn(h[v][2 * i], h[v][2 * i + 1]);
            *reinterpret_cast<uint4*>(static_cast<half*>(p.out) + row * p.out_pitch + g * 8) = r;
        }
    }
}

// Any width and any alignment: a row to a CTA, in shared memory, elements one by one.
template <bool kNorm, bool kCodes>
__global__ void __launch_bounds__(256) row_any_kernel(const __grid_constant__ RowParams p) {
    extern __shared__ float line[];
    __shared__ float warp_sums[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    float sum = 0.f;
    for (int i = tid; i < p.width; i += 256) {
        float h = __half2float(p.x[row * p.x_pitch + i]);
        if (p.skip) h += __half2float(p.skip[row * p.skip_pitch + i]);
        if (p.residual) p.residual[row * p.residual_pitch + i] = __float2half_rn(h);
        line[i] = h;
        sum = fmaf(h, h, sum);
    }
    float factor = 1.f;
    sum = warp_sum(sum);
    if (lane == 0) warp_sums[warp] = sum;
    __syncthreads();
    if constexpr (kNorm) factor = rsqrtf(warp_sum(lane < 8 ? warp_sums[lane] : 0.f) / (float)p.width + p.eps);
    for (int b = warp * kScaleBlock; b < p.width; b += 8 * kScaleBlock) {
        float y[4], top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = b + i * 32 + lane;
            y[i] = c < p.width ? line[c] : 0.f;
            if constexpr (kNorm) y[i] = c < p.width ? y[i] * factor * __half2float(p.gamma[c]) : 0.f;
            top = max_nan(top, fabsf(y[i]));
        }
        if constexpr (kCodes) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (lane == 0) p.scales[(long long)(b / kScaleBlock) * p.rows + row] = Scale(top).scale;
        }
        const Scale s(top);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = b + i * 32 + lane;
            if (c >= p.width) continue;
            if constexpr (kCodes) static_cast<uint8_t*>(p.out)[row * p.out_pitch + c] = (uint8_t)e4m3_pair(make_float2(quotient(y[i], s.scale, s.inverse), 0.f));
            else static_cast<half*>(p.out)[row * p.out_pitch + c] = __float2half_rn(y[i]);
        }
    }
}

template <bool kNorm, bool kSkip, bool kCodes>
cudaError_t launch_rows(const RowParams& p, cudaStream_t st) {
    // As few granules to a thread as leave a CTA 128 threads.
    const int granules = p.width / 8, v = granules <= 256 ? 1 : granules <= 512 ? 2 : 4;
    const int threads = ((granules + v - 1) / v + 31) / 32 * 32;
    const auto kernel = v == 1 ? row_kernel<1, kNorm, kSkip, kCodes> : v == 2 ? row_kernel<2, kNorm, kSkip, kCodes> : row_kernel<4, kNorm, kSkip, kCodes>;
    return launch_pdl(kernel, dim3((unsigned)p.rows), dim3(threads), 0, st, p);
}

template <bool kNorm, bool kCodes>
cudaError_t launch_any(const RowParams& p, cudaStream_t st) {
    const auto kernel = row_any_kernel<kNorm, kCodes>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxWidth * 4); });
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)p.rows), dim3(256), (size_t)p.width * 4, st, p);
}

bool granular(const void* a, long long pitch, int bytes) { return !a || (((reinterpret_cast<uintptr_t>(a) | (uintptr_t)(pitch * bytes)) & (uintptr_t)(8 * bytes - 1)) == 0); }

int rows_run(const RowParams& p, bool norm, cudaStream_t st, const char* where) {
    const bool codes = p.scales != nullptr;
    const bool vec = p.width % 8 == 0 && p.width <= 16384 && granular(p.x, p.x_pitch, 2) && granular(p.skip, p.skip_pitch, 2) && granular(p.residual, p.residual_pitch, 2) &&
                     granular(p.gamma, 0, 2) && granular(p.out, p.out_pitch, codes ? 1 : 2);
    cudaError_t e;
    if (!norm) e = vec ? launch_rows<false, false, true>(p, st) : launch_any<false, true>(p, st);
    else if (!vec) e = codes ? launch_any<true, true>(p, st) : launch_any<true, false>(p, st);
    else if (p.skip) e = codes ? launch_rows<true, true, true>(p, st) : launch_rows<true, true, false>(p, st);
    else e = codes ? launch_rows<true, false, true>(p, st) : launch_rows<true, false, false>(p, st);
    return cuda_status(e, where);
}

}  // namespace
}  // namespace et

extern "C" int et_skip_rmsnorm(const et_skip_rmsnorm_args* a) {
    using namespace et;
    ET_REQUIRE(a, "et_skip_rmsnorm: null pointer");
    ET_REQUIRE(a->rows >= 0, "et_skip_rmsnorm: negative size");
    ET_REQUIRE(a->width >= 1 && a->width <= kMaxWidth, "et_skip_rmsnorm: width must be 1 to 32768");
    ET_REQUIRE(a->eps > 0.f && a->eps <= 1.f, "et_skip_rmsnorm: eps must be above 0 and at most 1");
    if (a->rows == 0) return ET_OK;
    ET_REQUIRE(a->out && a->x && a->gamma, "et_skip_rmsnorm: null pointer");
    ET_REQUIRE(a->out_pitch >= a->width && a->x_pitch >= a->width && (!a->skip || a->skip_pitch >= a->width) && (!a->residual || a->residual_pitch >= a->width),
               "et_skip_rmsnorm: pitch below the width");
    ET_REQUIRE(a->residual != a->out, "et_skip_rmsnorm: residual and out are different results");
    // a result may lie where an operand lies, row for row
    const int out_bytes = a->scales ? 1 : 2;
    ET_REQUIRE((a->residual != a->x || a->residual_pitch == a->x_pitch) && (!a->residual || a->residual != a->skip || a->residual_pitch == a->skip_pitch),
               "et_skip_rmsnorm: in place the pitches must be equal");
    ET_REQUIRE((a->out != a->x || (out_bytes == 2 && a->out_pitch == a->x_pitch)) && (a->out != a->skip || (out_bytes == 2 && a->out_pitch == a->skip_pitch)),
               "et_skip_rmsnorm: in place out is fp16 and the pitches are equal");
    RowParams p;
    p.out = a->out; p.x = static_cast<const half*>(a->x); p.skip = static_cast<const half*>(a->skip); p.gamma = static_cast<const half*>(a->gamma);
    p.residual = static_cast<half*>(a->residual); p.scales = a->scales;
    p.out_pitch = a->out_pitch; p.x_pitch = a->x_pitch; p.skip_pitch = a->skip_pitch; p.residual_pitch = a->residual_pitch;
    p.rows = a->rows; p.width = a->width; p.eps = a->eps;
    return rows_run(p, true, static_cast<cudaStream_t>(a->stream), "et_skip_rmsnorm launch");
}

extern "C" int et_quantise_rows(const et_quantise_rows_args* a) {
    using namespace et;
    ET_REQUIRE(a, "et_quantise_rows: null pointer");
    ET_REQUIRE(a->rows >= 0, "et_quantise_rows: negative size");
    ET_REQUIRE(a->width >= 1 && a->width <= kMaxWidth, "et_quantise_rows: width must be 1 to 32768");
    if (a->rows == 0) return ET_OK;
    ET_REQUIRE(a->out && a->x && a->scales, "et_quantise_rows: null pointer");
    ET_REQUIRE(a->out != a->x, "et_quantise_rows: out may not be x");
    ET_REQUIRE(a->out_pitch >= a->width && a->x_pitch >= a->width, "et_quantise_rows: pitch below the width");
    RowParams p = {};
    p.out = a->out; p.x = static_cast<const half*>(a->x); p.scales = a->scales;
    p.out_pitch = a->out_pitch; p.x_pitch = a->x_pitch; p.rows = a->rows; p.width = a->width; p.eps = 1.f;
    return rows_run(p, false, static_cast<cudaStream_t>(a->stream), "et_quantise_rows launch");
}
