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
// sum is enough to move n by an ulp.  The Q8_0 form gives the codes and scales of fp64 arithmetic, whatever the
// row's split over threads: the sum of squares is in fp64, and n in fp32 decides only what its error (below
// 6 x 2^-24) cannot change.  A warp where a value lies within that of a border, or a block's maximum of
// one between two scales, or anything is not finite, does its eight values a thread again in fp64 (about
// one warp in ten).  8192 x 7168, bf16 + f32: 144 us against 100 of HBM; the 2-byte stores of the 34-byte blocks cost 10,
// the sum's conversions 3, the rest is the two phases of a row on two CTAs per SM.
//
// HBM bounds many rows (8192 x 7168, bf16 + f32 -> f32 + bf16: 106 us, 6.65 TB/s), one read's latency and the block's
// sum few (one row of 7168: 3.1 us).
#include "ck_launch.h"
#include "serve_common.cuh"

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
    const int32_t *live;  // NULL, or a row count: rows from it on take x as zero and leave res_out alone
};

CK_DEV void load_gain(const float *gain, uint32_t g, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(gain)[g * 2], b = reinterpret_cast<const float4 *>(gain)[g * 2 + 1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

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
// A row past the live ones is made zero after the loads: a test between them, though never true, kept them from being
// in flight together (8192 x 7168: 136 us for 106).
template <int VPT>
__global__ void __launch_bounds__(VPT == 1 ? 1024 : VPT == 2 ? 512 : 256) k_rmsnorm_add(const NormArgs p) {
    __shared__ float part[32];
    grid_dep_trigger_small();
    grid_dep_wait();
    const uint32_t nv = p.hidden >> 3;
    const uint64_t row = blockIdx.x;
    const bool pad = p.live && (int64_t)row >= *p.live;
    Raw8 rx[VPT], rr[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        if (g < nv) {
            rx[i] = load_raw8(p.x, row * p.x_stride + g * 8, p.x_type);
            if (p.res) rr[i] = load_raw8(p.res, row * p.res_stride + g * 8, p.res_type);
        }
    }
    float s[VPT][8];
    float acc = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        if (g < nv) {
            raw8_to_float(rx[i], p.x_type, s[i]);
            if (pad) {
#pragma unroll
                for (int j = 0; j < 8; ++j) s[i][j] = 0.0f;
            }
            if (p.res) {
                float r[8];
                raw8_to_float(rr[i], p.res_type, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[i][j] += r[j];
                if (p.res_out && !pad) store8(p.res_out, row * p.res_stride + g * 8, p.res_type, s[i]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) acc += s[i][j] * s[i][j];
        }
    }
    acc = block_sum(acc, part);
    const float inv = 1.0f / sqrtf(acc / (float)p.hidden + p.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        if (g < nv) {
            float gn[8], v[8];
            load_gain(p.gain, g, gn);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = s[i][j] * inv * gn[j];
            store8(p.out, row * p.out_stride + g * 8, p.out_type, v);
        }
    }
}

// The Q8_0 form.  A block of 32 values is four neighbouring threads' groups; hidden is a multiple of 32, so four
// neighbours are all live or all past the row.
template <int VPT>
__global__ void __launch_bounds__(VPT == 1 ? 1024 : VPT == 2 ? 512 : 256) k_rmsnorm_q8(const NormArgs p) {
    __shared__ double part[32];
    grid_dep_trigger_small();
    grid_dep_wait();
    const uint32_t nv = p.hidden >> 3;
    const uint64_t row = blockIdx.x;
    Raw8 rx[VPT], rr[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        rx[i].a = rx[i].b = rr[i].a = rr[i].b = make_uint4(0, 0, 0, 0);
        if (g < nv) {
            rx[i] = load_raw8(p.x, row * p.x_stride + g * 8, p.x_type);
            if (p.res) rr[i] = load_raw8(p.res, row * p.res_stride + g * 8, p.res_type);
        }
    }
    double acc = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        float x[8], r[8];
        raw8_to_float(rx[i], p.x_type, x);
        raw8_to_float(rr[i], p.res_type, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double v = p.res ? (double)x[j] + (double)r[j] : (double)x[j];
            acc += v * v;
            x[j] += r[j];
        }
        if (p.res_out && g < nv) store8(p.res_out, row * p.res_stride + g * 8, p.res_type, x);
    }
    acc = block_sum(acc, part);
    const double inv = 1.0 / sqrt(acc / (double)p.hidden + (double)p.eps);
    const float inv32 = (float)inv;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t g = threadIdx.x + i * blockDim.x;
        const bool live = g < nv;
        float x[8], r[8], gn[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        raw8_to_float(rx[i], p.x_type, x);
        raw8_to_float(rr[i], p.res_type, r);
        if (live) load_gain(p.gain, g, gn);
        float n[8], mx = 0.0f;
        bool unsure = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            n[j] = (x[j] + r[j]) * inv32 * gn[j];
            mx = fmaxf(mx, fabsf(n[j]));
            unsure |= n[j] != n[j];
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float q = mx / 127.0f;
        // the scale is sure where a relative step of 2^-21 either way rounds to it too
        __half d16 = __float2half_rn(q);
        const float d = __half2float(d16);
        unsure |= __half_as_ushort(__float2half_rn(q * (1.0f + 0x1p-21f))) !=
                  __half_as_ushort(__float2half_rn(q * (1.0f - 0x1p-21f)));
        unsure |= !(d > 0.0f && d < 1e30f);
        const float id = 1.0f / d;
        int code[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = n[j] * id, c = rintf(t);  // |t| <= 128: off by less than 128 x 6 x 2^-24 < 1e-4
            unsure |= fabsf(t - c) > 0.5f - 1e-4f;
            code[j] = max(-127, min(127, (int)c));
        }
        if (__any_sync(0xffffffffu, unsure && live)) {
            double m = 0, w[8];
            bool nan = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[j] = (p.res ? (double)x[j] + (double)r[j] : (double)x[j]) * inv * (double)gn[j];
                nan |= w[j] != w[j];
                m = fmax(m, fabs(w[j]));
            }
            if (nan) m = __longlong_as_double(0x7ff0000000000000ll);  // the block's scale says so
            m = fmax(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmax(m, __shfl_xor_sync(0xffffffffu, m, 2));
            d16 = __float2half_rn((float)(m / 127.0));
            const double dd = (double)__half2float(d16), idd = dd > 0 && dd < 1e30 ? 1.0 / dd : 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                code[j] = idd > 0 ? max(-127, min(127, __double2int_rn(w[j] * idd))) : 0;
        }
        if (live) {
            uint16_t *o = reinterpret_cast<uint16_t *>(static_cast<uint8_t *>(p.out) +
                                                       (row * (p.hidden >> 5) + (g >> 2)) * Q80_BYTES);
            if ((g & 3) == 0) o[0] = __half_as_ushort(d16);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[1 + (g & 3) * 4 + j] = (uint16_t)((code[2 * j] & 0xFF) | (code[2 * j + 1] & 0xFF) << 8);
        }
    }
}

template <int VPT>
cudaError_t launch_as(const NormArgs &a, uint32_t ntok, cudaStream_t s) {
    const uint32_t threads = (((a.hidden >> 3) + VPT - 1) / VPT + 31) / 32 * 32;
    if (a.out_type == T_Q8_0) return launch_pdl(k_rmsnorm_q8<VPT>, dim3(ntok), dim3(threads), 0, s, a);
    return a.live ? launch_pdl(k_rmsnorm_add<VPT>, dim3(ntok), dim3(threads), 0, s, a)
                  : launch_pdl(k_rmsnorm_add<VPT>, dim3(ntok), dim3(threads), 0, s, a);
}

int launch(const NormArgs &a, uint32_t ntok, cudaStream_t s) {
    const uint32_t nv = a.hidden >> 3;
    // groups per thread: one where few rows leave the SMs idle anyway (the row's latency counts), more
    // where rows queue up
    const bool few = ntok <= 2 * SMS;
    if (nv <= 1024 && (few || nv <= 128)) return (int)launch_as<1>(a, ntok, s);
    // the Q8_0 form computes more per value: more warps hide it better (8192 x 7168: 144 against 175 us)
    if (nv <= 512 || (nv <= 1024 && a.out_type == T_Q8_0)) return (int)launch_as<2>(a, ntok, s);
    if (nv <= 1024) return (int)launch_as<4>(a, ntok, s);
    return (int)launch_as<8>(a, ntok, s);
}

}  // namespace

int launch_rmsnorm_add(int x_type, const void *x, uint64_t x_stride, int res_type, const void *res, void *res_out,
                       uint64_t res_stride, const float *gain, int out_type, void *out, uint64_t out_stride,
                       uint32_t ntok, uint32_t hidden, float eps, cudaStream_t s, const int32_t *live) {
    if (live && out_type == T_Q8_0) return CK_ERR_ARG;
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
                        out_type, eps, live};
    return launch(a, ntok, s);
}

}  // namespace ck
