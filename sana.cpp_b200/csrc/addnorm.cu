// Residual addition and root-mean-square norm in one pass over a row:
//   h = x + r (rounded to r's type, the type the stream is held in),
//   y = h * rsqrt(sum(h^2) / C + eps) * (w + w0),
// written in fp32, bf16, or e4m3 with one scale per group of channels,
//   s = max(max|y| / 448, 2^-100), q = y / s.
// One block per row holds the row in registers, so that x and r are read once and h and y
// written once; the sum of squares is fp32, each thread's elements first, then a fixed tree over
// lanes and warps (the same bits every run). h is rounded before it is squared so that the norm is
// that of the stream a later reader sees; y is rounded once, at its store. Bound by HBM for many rows
// (38400 x 2304, bf16 + fp32 stream to e4m3 with a scale per 128: 163 to 172 us a call, 5.7 to 6.0 TB/s), by the launch for few.
#include <cuda_fp8.h>

#include "encoder.h"

namespace sana {
namespace {

constexpr float kE4M3Max = 448.0f;
constexpr float kScaleFloor = 7.888609052210118e-31f;  // 2^-100: its reciprocal stays finite

template <class T, int VEC>
__device__ __forceinline__ void load_row(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = to_f(p[0]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = f2_split(f2_from_bf2(w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

__device__ __forceinline__ uint32_t bf2_pack(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

template <class T, int VEC>
__device__ __forceinline__ void store_row(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        p[0] = from_f<T>(v[0]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(bf2_pack(v[0], v[1]), bf2_pack(v[2], v[3]), bf2_pack(v[4], v[5]),
                                                  bf2_pack(v[6], v[7]));
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN on either side stays
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

struct RowArgs {
    long long ldx, ldr, ldo;
    const float* weight;
    float* scale;
    int C, group, groups;
    float offset, eps;
};

// VEC channels per load (8: 16-byte bf16 and 2 x 16-byte fp32 vectors; 1: any alignment and
// width), PER loads per thread: channel (i * blockDim + tid) * VEC.
template <class TX, class TR, class TO, int VEC, int PER, bool RES>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(const TX* x, const TR* r, TR* sum, TO* out, RowArgs a) {
    constexpr bool kQuant = sizeof(TO) == 1;
    __shared__ float red[32];
    extern __shared__ unsigned int gmax[];  // E4M3: max|y| per group, as bits (they order as the values do, NaN on top)
    const long long row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const TX* xr = x + row * a.ldx;
    const TR* rr = RES ? r + row * a.ldr : nullptr;
    float h[PER][VEC];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = (i * blockDim.x + tid) * VEC;
        if (c < a.C) load_row<TX, VEC>(xr + c, h[i]);
    }
    if constexpr (RES) {
        float rv[PER][VEC];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * blockDim.x + tid) * VEC;
            if (c < a.C) load_row<TR, VEC>(rr + c, rv[i]);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] = to_f(from_f<TR>(h[i][j] + rv[i][j]));
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = (i * blockDim.x + tid) * VEC;
        if (c >= a.C) continue;
        if (RES && sum) store_row<TR, VEC>(sum + row * a.ldr + c, h[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) red[warp] = ss;
    if constexpr (kQuant) {
        for (int g = tid; g < a.groups; g += blockDim.x) gmax[g] = 0u;
    }
    __syncthreads();
    ss = lane < warps ? red[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = 1.0f / sqrtf(ss / static_cast<float>(a.C) + a.eps);

#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = (i * blockDim.x + tid) * VEC;
        if (c >= a.C) continue;
        if (a.weight) {
            float w[VEC];
            load_row<float, VEC>(a.weight + c, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] = h[i][j] * inv * (w[j] + a.offset);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[i][j] *= inv;
        }
        if constexpr (!kQuant) store_row<TO, VEC>(out + row * a.ldo + c, h[i]);
    }
    if constexpr (kQuant) {
        // Each load lies in one group (VEC divides the group). Consecutive lanes hold consecutive
        // channels, so lanes of one group first agree on their maximum; one of them adds it to the
        // group's shared word. The maximum does not depend on the order.
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * blockDim.x + tid) * VEC;
            const int g = c < a.C ? c / a.group : -1;
            float m = 0.f;
            if (c < a.C) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) m = max_nan(m, fabsf(h[i][j]));
            }
            const unsigned int peers = __match_any_sync(0xffffffffu, g);
            const unsigned int top = __reduce_max_sync(peers, __float_as_uint(m) & 0x7fffffffu);
            if (g >= 0 && lane == __ffs(peers) - 1) atomicMax(&gmax[g], top);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * blockDim.x + tid) * VEC;
            if (c >= a.C) continue;
            const int g = c / a.group;
            const float s = max_nan(__uint_as_float(gmax[g]) / kE4M3Max, kScaleFloor);
            // y / s in fp32 from the group's reciprocal and one residual (Markstein 1990): quotients that
            // fp32 holds come out exact, so that those midway between two e4m3 values go to the even one, which
            // the product alone can miss. Where s is infinite the residual is left at y, and finite y give 0.
            // 38400 x 2304, device time: 148.2 us, 146.9 with the product alone, 155.8 with divisions.
            const float inv_s = 1.0f / s, minus_s = s < INFINITY ? -s : 0.f;
            auto quotient = [&](float y) {
                const float q = y * inv_s;
                return fmaf(fmaf(q, minus_s, y), inv_s, q);
            };
            if (c == g * a.group) a.scale[row * a.groups + g] = s;
            TO* o = out + row * a.ldo + c;
            if constexpr (VEC == 1) {
                *reinterpret_cast<__nv_fp8_storage_t*>(o) = __nv_cvt_float_to_fp8(quotient(h[i][0]), __NV_SATFINITE, __NV_E4M3);
            } else {
                uint32_t w[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(quotient(h[i][4 * j]), quotient(h[i][4 * j + 1])),
                                                                 __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
                        make_float2(quotient(h[i][4 * j + 2]), quotient(h[i][4 * j + 3])), __NV_SATFINITE, __NV_E4M3);
                    w[j] = lo | (hi << 16);
                }
                *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
            }
        }
    }
}

template <class TX, class TR, class TO, bool RES>
void launch(const AddRmsNorm& p, int num_sms, cudaStream_t st) {
    RowArgs a;
    a.ldx = p.ldx;
    a.ldr = p.ldr;
    a.ldo = p.ldo;
    a.weight = p.weight;
    a.scale = p.scale;
    a.C = p.C;
    a.group = p.group && p.group < p.C ? p.group : p.C;
    a.groups = (p.C + a.group - 1) / a.group;
    a.offset = p.offset;
    a.eps = p.eps;
    const TX* x = static_cast<const TX*>(p.x);
    const TR* r = static_cast<const TR*>(p.residual);
    TR* sum = static_cast<TR*>(p.sum);
    TO* out = static_cast<TO*>(p.out);
    const size_t smem = sizeof(TO) == 1 ? static_cast<size_t>(a.groups) * 4 : 0;
    auto aligned = [](const void* q, long long ld, size_t size) {
        return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && (ld * static_cast<long long>(size)) % 16 == 0;
    };
    auto out_aligned = [&] {
        constexpr int kBytes = sizeof(TO) == 1 ? 8 : 16;  // the store's width
        return (reinterpret_cast<uintptr_t>(p.out) % kBytes) == 0 && (p.ldo * static_cast<long long>(sizeof(TO))) % kBytes == 0;
    };
    const bool vec = p.C % 8 == 0 && a.group % 8 == 0 && aligned(x, p.ldx, sizeof(TX)) && out_aligned() &&
                     (!RES || (aligned(r, p.ldr, sizeof(TR)) && aligned(sum, p.ldr, sizeof(TR)))) &&
                     (reinterpret_cast<uintptr_t>(p.weight) & 15) == 0;
    const unsigned grid = static_cast<unsigned>(p.rows);
    auto run = [&](auto* kernel, int block) {
        if (smem > 40960)  // beyond what a launch gets unasked: single channels as groups of wide rows
            SANA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        kernel<<<grid, block, smem, st>>>(x, r, sum, out, a);
    };
    auto threads = [&](int units, int per) { return (((units + per - 1) / per + 31) / 32) * 32; };
    if (vec) {
        const int units = p.C / 8;
        if (units <= 1024) {
            run(&add_rms_norm_kernel<TX, TR, TO, 8, 1, RES>, threads(units, 1));
        } else {
            run(&add_rms_norm_kernel<TX, TR, TO, 8, 2, RES>, threads(units, 2));
        }
    } else if (p.C <= 4096) {
        run(&add_rms_norm_kernel<TX, TR, TO, 1, 4, RES>, threads(p.C, 4));
    } else {
        run(&add_rms_norm_kernel<TX, TR, TO, 1, 16, RES>, threads(p.C, 16));
    }
    SANA_CUDA(cudaGetLastError());
}

template <class TX, class TR, bool RES>
void by_out(const AddRmsNorm& p, int num_sms, cudaStream_t st) {
    if (p.out_dtype == kF32) launch<TX, TR, float, RES>(p, num_sms, st);
    else if (p.out_dtype == kBf16) launch<TX, TR, bf16, RES>(p, num_sms, st);
    else launch<TX, TR, __nv_fp8_storage_t, RES>(p, num_sms, st);
}

template <class TX>
void by_residual(const AddRmsNorm& p, int num_sms, cudaStream_t st) {
    if (!p.residual) by_out<TX, TX, false>(p, num_sms, st);
    else if (p.r_dtype == kF32) by_out<TX, float, true>(p, num_sms, st);
    else by_out<TX, bf16, true>(p, num_sms, st);
}

}  // namespace

void add_rms_norm(const AddRmsNorm& p, int num_sms, cudaStream_t st) {
    if (p.rows == 0) return;
    if (p.x_dtype == kF32) by_residual<float>(p, num_sms, st);
    else by_residual<bf16>(p, num_sms, st);
}

}  // namespace sana
