// serve_common.cuh -- shared pieces of the serving kernels (norm_kernels.cu, kv_kernels.cu,
// attn_paged.cu, attn_chunk.cu): element types by their GGUF numbers, and 8-element
// loads and stores.
#pragma once
#include "ck_common.cuh"

namespace ck {

// GGUF type numbers, as everywhere in this library
constexpr int T_F32 = 0, T_F16 = 1, T_Q8_0 = 8, T_BF16 = 30;
constexpr uint32_t SMS = 148;  // SMs of a B200

__host__ __device__ inline int type_bytes(int t) { return t == T_F32 ? 4 : 2; }
inline bool float_type(int t) { return t == T_F32 || t == T_F16 || t == T_BF16; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Eight consecutive elements as loaded: 16 bytes of a 2-byte type, 32 of fp32.  Loading and
// converting are apart so that a thread's loads are all in flight before the first is used.
struct Raw8 {
    uint4 a, b;
};
CK_DEV Raw8 load_raw8(const void *base, uint64_t elem, int type) {
    Raw8 r;
    const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(base) + elem * (type == T_F32 ? 4 : 2));
    r.a = p[0];
    r.b = type == T_F32 ? p[1] : make_uint4(0, 0, 0, 0);
    return r;
}
CK_DEV void raw8_to_float(const Raw8 &r, int type, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == T_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else if (type == T_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
CK_DEV uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// two values rounded to nearest even in a 2-byte type
CK_DEV uint32_t pack2(int type, float lo, float hi) { return type == T_BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi); }
CK_DEV void store8(void *base, uint64_t elem, int type, const float (&v)[8]) {
    uint8_t *p = static_cast<uint8_t *>(base) + elem * (type == T_F32 ? 4 : 2);
    if (type == T_F32) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(type, v[0], v[1]), pack2(type, v[2], v[3]),
                                                   pack2(type, v[4], v[5]), pack2(type, v[6], v[7]));
    }
}

}  // namespace ck
