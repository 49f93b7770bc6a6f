// attn_paged.cu -- attention of few new tokens per request over a paged K/V cache (decode steps,
// short drafts, and every form the chunk kernel does not take).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  j over the visible keys
//
// in one pass over the keys with the running maximum and sum of each row.  The rows of a tile are 16
// (token, grouped query head) pairs that share a K/V head, so each K and V row is read once for all
// of them.  HBM bounds it: a decode step does 4 x rows flop per cache element.  One token over 131,072 (32 heads over 8,
// f16): 92 us, 5.8 TB/s, 89% of the measured copy rate; 64 ragged decodes of up to 8192 tokens 193 us
// (88%).  Short contexts are bound by latency: one token over 1000 with 56 heads in the f32 form 20 us, of which finding
// the work 2, the first keys 2, three units 5, joining warps and CTAs 4, the rest launch and skew.
//
// A CTA has four warps.  A unit is 64 keys; each warp takes 16 of them and has a ring of its own of
// STAGES x (16 K rows + 16 V rows) in shared memory, filled by 16-byte asynchronous copies whose
// page lookups run a unit ahead, so no warp waits for another until the item's end.  Ring and cursor run
// on across items.  S = Q K^T and O += P V run on mma.m16n8k16 (the 16 rows are one tile: the
// fifth-generation instructions start at 64), with fp32 accumulation; P goes from the first product's
// registers to the second's operands.
//
// With f32 queries and outputs the operands keep fp32's accuracy and range, and every product with a K or V element
// is exact in the accumulator.  bf16 caches: Q and P are split into three bf16 terms of 8 bits, each the rounding of
// the remainder.  f16 caches: into two tf32 terms of 11 bits, an f16 element being a tf32 value (64 ragged decodes of
// up to 8192 tokens 318 us; with three bf16 terms, each element the sum of two bf16 values, 377).  f16 terms would
// take half the products (246 us), but have no room for small weights and query elements: those under 2^-14 lose
// bits, those under 2^-25 are lost.  A remainder may be zero or negative, so infinities of V are kept out of every
// such product and added afterwards.  With 2-byte queries P is rounded once to the cache's type, an error of half an
// ulp of each weight: against 64 bits the outputs are off by 1.25 times what their own rounding alone gives (64 ragged
// decodes, bf16: 0.0021 of their norm for 0.0017; one token over 131,072, f16: 0.00028 for 0.00021).  f16 weights are taken times LIFT = 2^15 (they stay below
// 65504), so that only those under 2^-29 of their row's largest fall among f16's subnormals, where a weight is off by
// at most 2^-40 of the largest.
#include "attn_sched.cuh"

#include <type_traits>

namespace ck {
namespace attn {
namespace {

constexpr int TR = 16, KC = 64, WARPS = 4, WK = KC / WARPS;  // rows, keys per unit, warps, keys per warp
using S = Sched<TR, KC, false>;

// TERMS: 1 for 2-byte queries; for f32 ones three (bf16) or two (tf32, f16 caches)
template <int DP, int TERMS>
struct Few {
    static constexpr int ROW = DP * 2;  // bytes of a K or V row in shared memory
    static constexpr int STAGES = DP <= 64 ? 4 : 3;
    static constexpr int STAGE = 2 * WK * ROW;
    static constexpr int RING = WARPS * STAGES * STAGE;
    // the query tile (all terms), and after the last key two 16 x DP fp32 sums over two warps each
    static constexpr int QO = DP * 8 * TR;
    static_assert((TERMS == 2 ? 2 * DP * 4 : TERMS * ROW) <= DP * 8, "the query tile's terms");
    static constexpr int SMEM = RING + QO;
    static constexpr int CTAS = DP <= 64 ? 3 : DP <= 128 ? 2 : 1;  // per SM
};

CK_DEV void cp16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
CK_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
CK_DEV void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
CK_DEV void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
CK_DEV void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <int TYPE>
CK_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (TYPE == T_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the pair (lo, hi) rounded to bf16, and the remainders left in lo, hi
CK_DEV uint32_t split2(float &lo, float &hi) {
    const uint32_t w = pack_bf16x2(lo, hi);
    lo -= __uint_as_float(w << 16);
    hi -= __uint_as_float(w & 0xFFFF0000u);
    return w;
}
// v rounded to tf32, and the remainder left in v
CK_DEV float split_tf32(float &v) {
    uint32_t w;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(w) : "f"(v));
    const float t = __uint_as_float(w & 0xFFFFE000u);
    v -= t;
    return t;
}
// 16 x 8 by 8 x 8 in tf32; b: two f16 elements of a column.  A fragment's k runs over a thread's pairs in the order
// first elements, second elements, in a and b alike.
CK_DEV void mma_tf32(float (&c)[4], const float (&a)[4], uint32_t b) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&b));
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
                   "r"(__float_as_uint(a[3])), "r"(__float_as_uint(f.x)), "r"(__float_as_uint(f.y)));
}
// byte offset of element e (even) of row r in a query tile of tf32 terms: 16-byte pieces, swizzled so that the eight bytes
// of four rows by four neighbouring threads fall into different banks
template <int DP>
CK_DEV uint32_t tf32_at(int term, int r, int e) {
    return (uint32_t)((term * TR + r) * DP * 4 + ((((e >> 2) ^ ((r & 3) << 1)) << 4) | (e & 3) * 4));
}
// a pair of V elements with its infinities and NaNs replaced by zero
template <int TYPE>
CK_DEV uint32_t finite2(uint32_t w, bool &bad) {
    constexpr uint32_t M = TYPE == T_BF16 ? 0x7F80u : 0x7C00u;
    const bool l = (w & M) == M, h = (w >> 16 & M) == M;
    bad |= l | h;
    return (l ? 0u : w & 0xFFFFu) | (h ? 0u : w & 0xFFFF0000u);
}

// Joins the parts of an item that spans CTAs, in their order: a thread owns four neighbouring columns of a row and
// carries the running maximum and sum over the parts, whose loads depend on nothing.
template <int DP>
CK_DEV void join_parts(const AttnParams &p, const S::Joint &jt, const Pos &at, const Req &q, int rows) {
    constexpr int COLS = DP / 4;
    for (int i = threadIdx.x; i < rows * COLS; i += WARPS * 32) {
        const int r = i / COLS, col = i % COLS * 4;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 16
        for (int k = 0; k < jt.n; ++k) {
            const size_t s = jt.slot(k) * TR + r;
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.part_ml + s * 2));
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(p.part_o + s * DP + col));
            const float mn = fmaxf(m, ml.x), ref = mn == -INFINITY ? 0.0f : mn;
            const float a = ex2(m - ref), w = ex2(ml.x - ref);
            m = mn;
            l = l * a + w * ml.y;
            o.x = o.x * a + w * v.x;
            o.y = o.y * a + w * v.y;
            o.z = o.z * a + w * v.z;
            o.w = o.w * a + w * v.w;
        }
        const bool some = l > 0.0f || l != l;
        const float inv = some ? 1.0f / l : 0.0f;
        const int row = at.t * TR + r;
        const uint32_t tok = p.gd.div((uint32_t)row);
        const uint32_t head = at.h * p.gd.d + (row - tok * p.gd.d);
        if (col < (int)p.head_dim) {
            const uint64_t e = (uint64_t)(q.q0 + tok) * p.out_stride + (uint64_t)head * p.head_dim + col;
            if (p.io_type == T_F32)
                *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + e) =
                    make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            else
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + e) =
                    make_uint2(pack2(p.io_type, o.x * inv, o.y * inv), pack2(p.io_type, o.z * inv, o.w * inv));
        }
        if (p.lse && col == 0)
            p.lse[(uint64_t)(q.q0 + tok) * (p.n_kv * p.gd.d) + head] = some ? (m + log2f(l)) * LN2 : -INFINITY;
    }
}

template <int TYPE, int DP, int TERMS>
__global__ void __launch_bounds__(WARPS * 32, Few<DP, TERMS>::CTAS) k_attn_few(const __grid_constant__ AttnParams p) {
    using F = Few<DP, TERMS>;
    constexpr bool TF = TERMS == 2;
    constexpr float LIFT = TERMS == 1 && TYPE == T_F16 ? 32768.0f : 1.0f;
    static_assert(TERMS == 1 || TF == (TYPE == T_F16), "terms of the cache's type");
    constexpr int ROW = F::ROW, NS = F::STAGES, PIECES = DP / 8, COPIES = WK * PIECES / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ typename S::Shared sh;
    __shared__ float wm[WARPS][TR], wl[WARPS][TR];
    __shared__ int last_part;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(smem) + warp * NS * F::STAGE, qs = smem_u32(smem) + F::RING;
    float *osum = reinterpret_cast<float *>(smem + F::RING);
    grid_dep_trigger_small();
    grid_dep_wait();
    if (p.row_split == ATTN_NO_CHUNK && blockIdx.x == 0 && threadIdx.x == 0) *p.err = 0;  // the chunk form has no part
    long long U;
    int C;
    Pos pos;
    Geo geo;
    if (!S::find(p, sh, (int)gridDim.x, (int)blockIdx.x, U, C, pos, geo)) return;
    const long long u0 = S::start(U, C, blockIdx.x);
    const int n = (int)(S::start(U, C, blockIdx.x + 1) - u0);
    typename S::Items use, fill;
    if (!use.set(p, sh, n, u0)) return;
    fill = use;
    int fill_c = fill.c0;
    bool to_fill = true;

    // lane l < 16 looks up key l of the warp's next 16: its element offset, or -1 to fill with zeros
    // (past the tile's last key, so that what the page holds there never meets a product)
    const auto lookup = [&]() -> int64_t {
        const int j = fill.g.lo + fill_c * KC + warp * WK + (lane & 15);
        if (j >= fill.g.hi) return -1;
        const int64_t at = key_offset(p, fill.at.r, j);
        return at < 0 ? -1 : at + (int64_t)(fill.at.h * p.head_stride);
    };
    const auto copy_in = [&](int stage, int64_t off) {
        const uint32_t base = ring + stage * F::STAGE;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int idx = i * 32 + lane, row = idx / PIECES, c = idx % PIECES;
            const int64_t at = __shfl_sync(0xffffffffu, off, row);
            const bool live = at >= 0 && c * 8 < (int)p.head_dim;
            const int64_t e = live ? at + c * 8 : 0;
            const uint32_t dst = base + row * ROW + ((c ^ (row & 7)) << 4);
            cp16(dst, static_cast<const uint16_t *>(p.k) + e, live);
            cp16(dst + WK * ROW, static_cast<const uint16_t *>(p.v) + e, live);
        }
    };
    int filled = 0;
    int64_t off = lookup();
    const auto fill_next = [&]() {
        if (to_fill) {
            copy_in(filled % NS, off);
            ++filled;
            if (++fill_c == fill.c1) {
                to_fill = fill.next(p);
                fill_c = 0;
            }
            if (to_fill) off = lookup();
        }
        cp_commit();  // an empty group past the end keeps the count of groups in step
    };
    for (int i = 0; i < NS - 1; ++i) fill_next();

    int i = 0;  // units done
    for (int segment = 0;; ++segment) {
        const int rows = use.q.nq * (int)p.gd.d, row0 = use.at.t * TR;
        float o[DP / 8][4];
        float m[2], l[2];
        int row_lo[2], row_hi[2];
        int all_lo, all_hi;  // keys [all_lo, all_hi) every row of the tile sees
        bool bad = false;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
        {
            // the query tile: eight threads per row
            const int r = threadIdx.x >> 3, part = threadIdx.x & 7, row = row0 + r;
            const bool live = row < rows;
            const uint32_t tok = p.gd.div((uint32_t)(live ? row : 0));
            const uint32_t head = use.at.h * p.gd.d + ((live ? row : 0) - tok * p.gd.d);
            const uint64_t at = (uint64_t)(use.q.q0 + tok) * p.q_stride + (uint64_t)head * p.head_dim;
            if constexpr (TERMS == 1) {
#pragma unroll
                for (int c = part; c < PIECES; c += 8) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (live && c * 8 < (int)p.head_dim)
                        w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + at + c * 8);
                    *reinterpret_cast<uint4 *>(smem + F::RING + r * ROW + ((c ^ (r & 7)) << 4)) = w;
                }
            } else {
                float v[DP / 64][8];
#pragma unroll
                for (int k = 0; k < DP / 64; ++k) {
                    const int c = part + 8 * k;
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[k][e] = 0.0f;
                    if (live && c * 8 < (int)p.head_dim) raw8_to_float(load_raw8(p.q, at + c * 8, T_F32), T_F32, v[k]);
                }
#pragma unroll
                for (int term = 0; term < TERMS; ++term)
#pragma unroll
                    for (int k = 0; k < DP / 64; ++k) {
                        const int c = part + 8 * k;
                        if constexpr (TF) {
#pragma unroll
                            for (int e = 0; e < 8; e += 4)
                                *reinterpret_cast<float4 *>(smem + F::RING + tf32_at<DP>(term, r, c * 8 + e)) =
                                    make_float4(split_tf32(v[k][e]), split_tf32(v[k][e + 1]), split_tf32(v[k][e + 2]),
                                                split_tf32(v[k][e + 3]));
                            continue;
                        }
                        uint4 w;
                        w.x = split2(v[k][0], v[k][1]);
                        w.y = split2(v[k][2], v[k][3]);
                        w.z = split2(v[k][4], v[k][5]);
                        w.w = split2(v[k][6], v[k][7]);
                        *reinterpret_cast<uint4 *>(smem + F::RING + term * TR * ROW + r * ROW + ((c ^ (r & 7)) << 4)) = w;
                    }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                m[k] = -INFINITY;
                l[k] = 0.0f;
                row_limits(p, use.q, min(row0 + (lane >> 2) + 8 * k, rows - 1), row_lo[k], row_hi[k]);
            }
            int dummy;
            row_limits(p, use.q, row0, dummy, all_hi);
            row_limits(p, use.q, min(row0 + TR, rows) - 1, all_lo, dummy);
            __syncthreads();
        }
        for (int c = use.c0; c < use.c1; ++c, ++i) {
            cp_wait<NS - 2>();
            __syncwarp();
            fill_next();
            const int j0 = use.g.lo + c * KC + warp * WK;
            if (j0 >= use.g.hi) continue;
            const uint32_t kb = ring + (i % NS) * F::STAGE, vb = kb + WK * ROW;
            // even and odd steps into sums of their own: half the chain of dependent products
            float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, s1[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll 2
            for (int ks = 0; ks < DP / 16; ++ks) {
                float(&sk)[2][4] = (ks & 1) ? s1 : s;
                uint32_t b[4];
                {  // keys 0-7 | 8-15 by the 16 dims of this step
                    const int key = (lane & 7) + ((lane >> 4) << 3), c = ks * 2 + ((lane >> 3) & 1);
                    ldsm4(kb + key * ROW + ((c ^ (key & 7)) << 4), b);
                }
#pragma unroll
                for (int term = 0; term < TERMS; ++term) {
                    if constexpr (TF) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int r = lane >> 2, e = ks * 16 + x * 8 + (lane & 3) * 2;
                            const float2 u = *reinterpret_cast<const float2 *>(smem + F::RING + tf32_at<DP>(term, r, e));
                            const float2 w = *reinterpret_cast<const float2 *>(smem + F::RING + tf32_at<DP>(term, r + 8, e));
                            const float a[4] = {u.x, w.x, u.y, w.y};
                            mma_tf32(sk[0], a, b[x]);
                            mma_tf32(sk[1], a, b[2 + x]);
                        }
                        continue;
                    }
                    uint32_t a[4];
                    const int r = lane & 15, c = ks * 2 + (lane >> 4);
                    ldsm4(qs + term * TR * ROW + r * ROW + ((c ^ (r & 7)) << 4), a);
                    mma<TYPE>(sk[0], a, b[0], b[1]);
                    mma<TYPE>(sk[1], a, b[2], b[3]);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] += s1[t][e];
            const bool partial = j0 < all_lo || j0 + WK > all_hi;  // some row does not see some key
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float &x = s[t][2 * k + e];
                        x *= p.scale_log2;
                        if (partial) {
                            const int j = j0 + t * 8 + (lane & 3) * 2 + e;
                            if (j < row_lo[k] || j >= row_hi[k]) x = -INFINITY;
                        }
                    }
                float mx = fmaxf(fmaxf(s[0][2 * k], s[0][2 * k + 1]), fmaxf(s[1][2 * k], s[1][2 * k + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[k], mx);
                const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: every weight below is 0
                const float al = ex2(m[k] - ref);
                m[k] = mn;
                l[k] *= al;
                if (al != 1.0f) {
#pragma unroll
                    for (int d = 0; d < DP / 8; ++d) {
                        o[d][2 * k] *= al;
                        o[d][2 * k + 1] *= al;
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float &x = s[t][2 * k + e];
                        x = ex2(x - ref);
                        l[k] += x;
                    }
            }
            if constexpr (TF) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {  // eight keys, by the 32 dims of a step
                    float a[TERMS][4];
#pragma unroll
                    for (int term = 0; term < TERMS; ++term)
#pragma unroll
                        for (int x = 0; x < 4; ++x) a[term][x] = split_tf32(s[t][(x & 1) * 2 + (x >> 1)]);
#pragma unroll
                    for (int dt = 0; dt < DP / 32; ++dt) {
                        uint32_t b[4];
                        const int key = t * 8 + (lane & 7), c = dt * 4 + (lane >> 3);
                        ldsm4t(vb + key * ROW + ((c ^ (key & 7)) << 4), b);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            b[x] = finite2<TYPE>(b[x], bad);
#pragma unroll
                            for (int term = 0; term < TERMS; ++term) mma_tf32(o[4 * dt + x], a[term], b[x]);
                        }
                    }
                }
                continue;
            }
            uint32_t a[TERMS][4];
#pragma unroll
            for (int term = 0; term < TERMS; ++term)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float &lo = s[x >> 1][(x & 1) * 2], &hi = s[x >> 1][(x & 1) * 2 + 1];
                    a[term][x] = TERMS > 1 ? split2(lo, hi) : pack2(TYPE, lo * LIFT, hi * LIFT);
                }
#pragma unroll
            for (int dt = 0; dt < DP / 16; ++dt) {
                uint32_t b[4];
                const int key = (lane & 7) + (((lane >> 3) & 1) << 3), c = dt * 2 + (lane >> 4);
                ldsm4t(vb + key * ROW + ((c ^ (key & 7)) << 4), b);
                if (TERMS > 1 || partial) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) b[x] = finite2<TYPE>(b[x], bad);
                }
#pragma unroll
                for (int term = 0; term < TERMS; ++term) {
                    mma<TYPE>(o[2 * dt], a[term], b[0], b[1]);
                    mma<TYPE>(o[2 * dt + 1], a[term], b[2], b[3]);
                }
            }
        }
        {
            // join the warps under their common maximum
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
                l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
                if ((lane & 3) == 0) {
                    wm[warp][(lane >> 2) + 8 * k] = m[k];
                    wl[warp][(lane >> 2) + 8 * k] = l[k];
                }
            }
            const bool any_bad = __syncthreads_or(bad);
            float f[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = (lane >> 2) + 8 * k;
                float mm = wm[0][r];
                for (int w = 1; w < WARPS; ++w) mm = fmaxf(mm, wm[w][r]);
                f[k] = ex2(m[k] - (mm == -INFINITY ? 0.0f : mm)) * (1.0f / LIFT);
            }
            // warps 0 and 1 lay their sums down, 2 and 3 add theirs to them
#pragma unroll
            for (int pass = 0; pass < 2; ++pass) {
                if ((warp >> 1) == pass) {
#pragma unroll
                    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float2 *at = reinterpret_cast<float2 *>(osum + ((warp & 1) * TR + (lane >> 2) + 8 * k) * DP +
                                                                    d * 8 + (lane & 3) * 2);
                            float2 v = make_float2(o[d][2 * k] * f[k], o[d][2 * k + 1] * f[k]);
                            if (pass) v.x += at->x, v.y += at->y;
                            *at = v;
                        }
                }
                __syncthreads();
            }
            const bool whole = use.whole();
            float *po = p.part_o + ((size_t)blockIdx.x * 2 + (segment ? 1 : 0)) * TR * DP;
            float *pm = p.part_ml + ((size_t)blockIdx.x * 2 + (segment ? 1 : 0)) * TR * 2;
            // eight threads per row, as for the queries
            const int r = threadIdx.x >> 3, part = threadIdx.x & 7, row = row0 + r;
            if (row < rows) {
                float mm = wm[0][r];
                for (int w = 1; w < WARPS; ++w) mm = fmaxf(mm, wm[w][r]);
                const float ref = mm == -INFINITY ? 0.0f : mm;
                float ll = 0.0f;
                for (int w = 0; w < WARPS; ++w) ll += wl[w][r] * ex2(wm[w][r] - ref);
                int lo, hi;
                row_limits(p, use.q, row, lo, hi);
                const uint32_t tok = p.gd.div((uint32_t)row);
                const uint32_t head = use.at.h * p.gd.d + (row - tok * p.gd.d);
                const float inv = whole ? (ll > 0.0f || ll != ll ? 1.0f / ll : 0.0f) : 1.0f;
                for (int c = part; c * 8 < (int)p.head_dim; c += 8) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = (osum[r * DP + c * 8 + e] + osum[(TR + r) * DP + c * 8 + e]) * inv;
                        if (any_bad)  // TERMS > 1: every step's V was cleaned
                            v[e] += nonfinite_v(p, use.at.r, use.at.h, c * 8 + e, use.g.lo + use.c0 * KC,
                                                min(use.g.lo + use.c1 * KC, use.g.hi), WK, TERMS > 1 ? 0x7fffffff : all_lo,
                                                all_hi, lo, hi);
                    }
                    if (whole)
                        store8(p.out, (uint64_t)(use.q.q0 + tok) * p.out_stride + (uint64_t)head * p.head_dim + c * 8,
                               p.io_type, v);
                    else
                        store8(po, (uint64_t)r * DP + c * 8, T_F32, v);
                }
                if (part == 0) {
                    if (!whole) {
                        pm[r * 2] = mm;
                        pm[r * 2 + 1] = ll;
                    } else if (p.lse) {
                        p.lse[(uint64_t)(use.q.q0 + tok) * (p.n_kv * p.gd.d) + head] =
                            ll > 0.0f || ll != ll ? (mm + log2f(ll)) * LN2 : -INFINITY;
                    }
                }
            }
            if (!whole) {
                // the part is out; whoever brings the item's last one joins them all
                const typename S::Joint jt = S::joint(use, U, C);
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) {
                    const bool last = atomicAdd(p.arrived + jt.cta, 1) == jt.n - 1;
                    if (last) p.arrived[jt.cta] = 0;
                    last_part = last;
                }
                __syncthreads();
                if (last_part) {
                    __threadfence();
                    join_parts<DP>(p, jt, use.at, use.q, min(rows - row0, TR));
                }
            }
        }
        if (!use.next(p)) break;
        __syncthreads();
    }
    cp_wait<0>();
}

template <int TYPE, int DP, int TERMS>
int launch(AttnParams p, cudaStream_t s) {
    using F = Few<DP, TERMS>;
    static unsigned long long done = 0;
    if (attr_pending(done)) {
        cudaError_t e = cudaFuncSetAttribute(k_attn_few<TYPE, DP, TERMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
        if (e != cudaSuccess) return (int)e;
        attr_mark(done);
    }
    const uint32_t grid = SMS * F::CTAS;
    p.part_ml = p.part_o + (size_t)grid * 2 * TR * DP;
    return (int)launch_pdl(k_attn_few<TYPE, DP, TERMS>, dim3(grid), dim3(WARPS * 32), F::SMEM, s, p);
}
template <int TYPE, int DP>
int launch_terms(const AttnParams &p, cudaStream_t s) {
    return p.io_type == T_F32 ? launch<TYPE, DP, TYPE == T_BF16 ? 3 : 2>(p, s) : launch<TYPE, DP, 1>(p, s);
}
template <int TYPE>
int launch_dim(const AttnParams &p, cudaStream_t s) {
    if (p.head_dim <= 64) return launch_terms<TYPE, 64>(p, s);
    if (p.head_dim <= 128) return launch_terms<TYPE, 128>(p, s);
    return launch_terms<TYPE, 256>(p, s);
}

}  // namespace
}  // namespace attn

size_t attn_few_workspace_bytes(uint32_t head_dim) {
    const size_t dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256, ctas = dp == 64 ? 3 : dp == 128 ? 2 : 1;
    return SMS * ctas * 2 * attn::TR * (dp + 2) * 4;
}

int launch_attn_few(const AttnParams &p, cudaStream_t s) {
    return p.cache_type == T_BF16 ? attn::launch_dim<T_BF16>(p, s) : attn::launch_dim<T_F16>(p, s);
}

}  // namespace ck
