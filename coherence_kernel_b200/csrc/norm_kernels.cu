// norm_kernels.cu -- RMS norm with the residual's addition, one pass over the row.
//
//   s[i]   = x[i] + res[i]                     (s = x without a residual)
//   res_out[i] = s[i] rounded to the residual's type
//   n[i]   = s[i] / sqrt(mean(s^2) + eps) * gain[i]
//   out[i] = n[i] rounded to f32 / bf16 / f16, or GGUF Q8_0: per 32 values d = f16(f32(max|n| / 127))
//            and codes clamp(round(n / d)) in -127..127
//
// The row's sum of squares is taken from the unrounded s, in fp32: per-thread sums, then the lanes
// of a warp and the warps in a fixed order, so results do not depend on timing.
//
// Q8_0 codes flip where n / d lies next to the border of two codes, and a different order of the
// sum is enough to move n by an ulp.  The Q8_0 form therefore takes s, the sum of squares and n in
// fp64: the codes are the definition's, whatever the row's split over threads.
//
// HBM bounds many rows (8192 x 7168, bf16 + f32 -> f32 + bf16: 106 us, 6.65 TB/s), one read's latency and the block's
// sum few (one row of 7168: 3.1 us).
#include "ck_launch.h"
#include "serve_common.cuh"

#include <type_traits>

namespace ck {
namespace {

struct NormArgs {
    const void *x, *res;
    void *res_out, *out;
    const float *gain;
    uint64_t x_stride, res_stride, out_stride;
    uint32_t hidden;
    int x_type, res_type, out_type;
    float eps;
};

template <typename F>
CK_DEV F block_sum(F v, F *part) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int nw = blockDim.x >> 5;
    if (nw == 1) return v;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    // every warp adds the partials in the same order
    F t = (int)(threadIdx.x & 31) < nw ? part[threadIdx.x & 31] : F(0);
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

// One CTA per row; a thread owns VPT groups of eight consecutive elements, blockDim.x groups apart,
// held in registers between the sum and the output.
template <int VPT, bool Q8>
__global__ void __launch_bounds__(VPT == 1 ? 1024 : VPT == 2 ? 512 : 256) k_rmsnorm_add(const NormArgs p) {
    using F = typename std::conditional<Q8, double, float>::type;
    __shared__ F part[32];
    grid_dep_trigger_small();
    grid_dep_wait();
    const uint32_t nv = p.hidden >> 3;
    const uint64_t row = blockIdx.x;
    Raw8 rx[VPT], rr[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        if (g < nv) {
            rx[i] = load_raw8(p.x, row * p.x_stride + g * 8, p.x_type);
            if (p.res) rr[i] = load_raw8(p.res, row * p.res_stride + g * 8, p.res_type);
        }
    }
    F s[VPT][8];
    F acc = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        if (g < nv) {
            float v[8], r[8];
            raw8_to_float(rx[i], p.x_type, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[i][j] = v[j];
            if (p.res) {
                raw8_to_float(rr[i], p.res_type, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[i][j] += (F)r[j];
                if (p.res_out) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = (float)s[i][j];
                    store8(p.res_out, row * p.res_stride + g * 8, p.res_type, v);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) acc += s[i][j] * s[i][j];
        }
    }
    acc = block_sum(acc, part);
    const F inv = F(1) / sqrt(acc / (F)p.hidden + (F)p.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        const bool live = g < nv;
        if constexpr (!Q8) {
            if (live) {
                const float4 g0 = reinterpret_cast<const float4 *>(p.gain)[g * 2];
                const float4 g1 = reinterpret_cast<const float4 *>(p.gain)[g * 2 + 1];
                const float gn[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = s[i][j] * inv * gn[j];
                store8(p.out, row * p.out_stride + g * 8, p.out_type, v);
            }
        } else {
            // a block of 32 values is four neighbouring threads' groups; hidden is a multiple of 32, so
            // four neighbours are all live or all past the row
            double mx = 0;
            if (live) {
                const float4 g0 = reinterpret_cast<const float4 *>(p.gain)[g * 2];
                const float4 g1 = reinterpret_cast<const float4 *>(p.gain)[g * 2 + 1];
                const float gn[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
                bool nan = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    s[i][j] = s[i][j] * inv * (double)gn[j];
                    nan |= s[i][j] != s[i][j];
                    mx = fmax(mx, fabs(s[i][j]));
                }
                if (nan) mx = __longlong_as_double(0x7ff0000000000000ll);  // the block's scale says so
            }
            mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (live) {
                const __half d16 = __float2half_rn((float)(mx / 127.0));
                const double d = (double)__half2float(d16);
                const double id = d > 0 && d < 1e30 ? 1.0 / d : 0.0;
                uint32_t code[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    code[j] = (uint32_t)(id > 0 ? max(-127, min(127, __double2int_rn(s[i][j] * id))) : 0) & 0xFFu;
                uint16_t *o = reinterpret_cast<uint16_t *>(static_cast<uint8_t *>(p.out) +
                                                           (row * (p.hidden >> 5) + (g >> 2)) * Q80_BYTES);
                if ((g & 3) == 0) o[0] = __half_as_ushort(d16);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[1 + (g & 3) * 4 + j] = (uint16_t)(code[2 * j] | code[2 * j + 1] << 8);
            }
        }
    }
}

template <bool Q8>
int launch(const NormArgs &a, uint32_t ntok, cudaStream_t s) {
    const uint32_t nv = a.hidden >> 3;
    const auto threads = [&](uint32_t vpt) { return ((nv + vpt - 1) / vpt + 31) / 32 * 32; };
    // groups per thread: one where few rows leave the SMs idle anyway (the row's latency counts), more
    // where rows queue up
    const bool few = ntok <= 2 * SMS;
    cudaError_t e;
    if (nv <= 1024 && (few || nv <= 128))
        e = launch_pdl(k_rmsnorm_add<1, Q8>, dim3(ntok), dim3(threads(1)), 0, s, a);
    else if (nv <= 512)
        e = launch_pdl(k_rmsnorm_add<2, Q8>, dim3(ntok), dim3(threads(2)), 0, s, a);
    else if (nv <= 1024)
        e = launch_pdl(k_rmsnorm_add<4, Q8>, dim3(ntok), dim3(threads(4)), 0, s, a);
    else
        e = launch_pdl(k_rmsnorm_add<8, Q8>, dim3(ntok), dim3(threads(8)), 0, s, a);
    return (int)e;
}

}  // namespace

int launch_rmsnorm_add(int x_type, const void *x, uint64_t x_stride, int res_type, const void *res, void *res_out,
                       uint64_t res_stride, const float *gain, int out_type, void *out, uint64_t out_stride,
                       uint32_t ntok, uint32_t hidden, float eps, cudaStream_t s) {
    if (!float_type(x_type) || (res && !float_type(res_type)) || (out_type != T_Q8_0 && !float_type(out_type)))
        return CK_ERR_ARG;
    if (hidden == 0 || hidden % (out_type == T_Q8_0 ? 32 : 8) || hidden > 16384) return CK_ERR_SHAPE;
    if (ntok == 0) return 0;
    if (ntok > 0x7fffffffu) return CK_ERR_SHAPE;
    if (!x || !gain || !out || (res_out && !res)) return CK_ERR_ARG;
    if (!aligned16(x) || !aligned16(res) || !aligned16(res_out) || !aligned16(gain) ||
        (reinterpret_cast<uintptr_t>(out) & (out_type == T_Q8_0 ? 1 : 15)))
        return CK_ERR_ARG;
    if (x_stride < hidden || x_stride % 8 || (res && (res_stride < hidden || res_stride % 8)) ||
        (out_type != T_Q8_0 && (out_stride < hidden || out_stride % 8)))
        return CK_ERR_ARG;
    const NormArgs a = {x, res, res_out, out, gain, x_stride, res_stride, out_stride, hidden, x_type, res_type,
                        out_type, eps};
    return out_type == T_Q8_0 ? launch<true>(a, ntok, s) : launch<false>(a, ntok, s);
}

}  // namespace ck
