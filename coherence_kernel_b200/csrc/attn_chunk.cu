// attn_chunk.cu -- attention of many rows (long chunks of new tokens, or many heads over one K/V head) over
// the paged cache, on the fifth-generation tensor cores.
//
// The same one-pass softmax as attn_paged.cu with tiles of 256 rows and units of 128 keys.  One CTA per
// SM of four warpgroups:
//   0, 1  softmax: each owns 128 rows, a thread one row.  Reads its scores from tensor memory (all 128 of
//         a unit in registers), masks, keeps maximum and sum, and writes P as bf16 / f16 pairs over the
//         scores it came from -- the A operand of the second product never leaves tensor memory
//   2     loader: K and V rows by 16-byte asynchronous copies (each row's page looked up by one lane a unit
//         ahead, so any page size and stride works) into a ring of four 128-key tiles in the 128-byte-swizzle
//         layout; the query tile at each item's start
//   3     one warp issues the products: S_t = Q_t K^T (both operands in shared memory) and
//         O_t += P_t V (P in tensor memory, V as an N-major B operand straight from its row layout)
// Tensor memory: S_0 S_1 O_0 O_1, 128 columns each.  The issue order PV_0(i) S_0(i+1) PV_1(i) S_1(i+1) keeps the
// tensor core on one half while the other half's softmax runs; S_t(i+1) may follow PV_t(i) unwaited, since
// one thread's products execute in order.
//
// O is rescaled only when a row's maximum has grown by more than 8 (in log2 units) since the maximum
// its weights refer to: weights stay below 2^8, exactly representable scaling, and most units skip the
// round trip of O through registers.  P is rounded once to the cache's type (half an ulp of each weight,
// below the output's own rounding); scores, sums and O are fp32.
//
// Bound: the tensor core (4 x 128 x 128 x 128 multiply-adds, 2048 cycles per unit) and the exponentials (2 x 128
// x 128 at 16 per cycle: 2048 cycles) alike.
#include "attn_sched.cuh"

namespace ck {
namespace attn {
namespace {

constexpr int TR = 256, KC = 128;
using S = Sched<TR, KC, true>;
constexpr int NTHREADS = 512;
constexpr float GROW = 8.0f;  // log2 growth of a row's maximum that makes O rescale

template <int DP>
struct Chunk {
    static constexpr int HALVES = DP / 64;             // 128-byte-wide column halves of a tile
    static constexpr int TILE = KC * DP * 2;           // a K or V tile; also 128 query rows
    static constexpr int STAGES = 4;
    static constexpr int Q_OFF = 0, RING_OFF = 2 * TILE, BAR_OFF = RING_OFF + STAGES * TILE;
    static constexpr int SMEM = BAR_OFF + 256 + 1024;  // + alignment of the tiles
    static_assert(SMEM <= 227 * 1024, "shared memory");
};
// mbarriers
struct Bars {
    uint64_t full[4], empty[4], q_full, q_empty, s_full[2], p_full[2], o_full[2], done;
};
// tensor memory: scores (and P over them) of the two halves, then their outputs
CK_DEV uint32_t s_col(int t) { return (uint32_t)t * 128; }
CK_DEV uint32_t o_col(int t) { return 256 + (uint32_t)t * 128; }
// 128-row halves of tile t of a request that hold rows
CK_DEV int halves(const AttnParams &p, const Req &q, int t) { return q.nq * (int)p.gd.d - t * TR > 128 ? 2 : 1; }

CK_DEV void cp16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
CK_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
CK_DEV void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int N>
CK_DEV void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
CK_DEV void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
CK_DEV bool elect_one() {
    uint32_t pred = 0;
    asm volatile("{\n .reg .b32 %%rx;\n .reg .pred %%px;\n elect.sync %%rx|%%px, %1;\n selp.u32 %0, 1, 0, %%px;\n}"
                 : "=r"(pred)
                 : "r"(0xffffffffu));
    return pred != 0;
}
// Instruction descriptor: 16-bit inputs -> fp32, A K-major, B K-major or (tb) N-major, M x N.
__host__ __device__ constexpr uint32_t idesc16(int type, int M, int N, int tb) {
    const uint32_t f = type == T_BF16 ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)tb << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// N-major, 128-byte swizzle: 64 columns x 8 k-rows are 1024 bytes (row pitch 128), the next 8 k-rows
// 1024 bytes on, the next 64 columns `half` bytes on.
CK_DEV uint64_t sdesc_n_sw128(uint32_t addr, uint32_t half) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFF);
    d |= (uint64_t)((half >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
template <int TYPE>
CK_DEV uint32_t finite2(uint32_t w, bool &bad) {
    constexpr uint32_t M = TYPE == T_BF16 ? 0x7F80u : 0x7C00u;
    const bool l = (w & M) == M, h = (w >> 16 & M) == M;
    bad |= l | h;
    return (l ? 0u : w & 0xFFFFu) | (h ? 0u : w & 0xFFFF0000u);
}
// whether some row of the item does not see some key of the unit at j0 (its V is then cleaned of infinities and NaNs)
CK_DEV void item_limits(const AttnParams &p, const Req &q, int t, int &all_lo, int &all_hi) {
    const int rows = q.nq * (int)p.gd.d;
    int dummy;
    row_limits(p, q, t * TR, dummy, all_hi);
    row_limits(p, q, min(t * TR + TR, rows) - 1, all_lo, dummy);
}

template <int TYPE, int DP>
__global__ void __launch_bounds__(NTHREADS, 1) k_attn_chunk(const AttnParams p) {
    using F = Chunk<DP>;
    constexpr int PIECES = DP / 8;           // 16-byte pieces of a row
    constexpr int ROWS_PER = 32 / PIECES;    // rows one warp instruction copies
    constexpr int NS = F::STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ typename S::Shared sh;
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t poison[8];  // item number + 1 of an item whose V was cleaned, by item modulo 8
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    Bars *bar = reinterpret_cast<Bars *>(smem + F::BAR_OFF);
    const uint32_t sbase = smem_u32(smem);
    const int wg = threadIdx.x >> 7, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_trigger_small();
    grid_dep_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.err = 0;
    long long U;
    int C;
    Pos pos;
    Geo geo;
    if (!S::find(p, sh, (int)gridDim.x, (int)blockIdx.x, U, C, pos, geo)) return;
    const int n = (int)(S::start(U, C, blockIdx.x + 1) - S::start(U, C, blockIdx.x));
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bar->full[i], 128);
            mbar_init(&bar->empty[i], 1);
        }
        mbar_init(&bar->q_full, 128);
        mbar_init(&bar->q_empty, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&bar->s_full[t], 1);
            mbar_init(&bar->p_full[t], 128);
            mbar_init(&bar->o_full[t], 1);
        }
        mbar_init(&bar->done, 1);
        fence_barrier_init();
    }
    if (threadIdx.x < 8) poison[threadIdx.x] = 0;
    if (warp == 12) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (wg == 2) {
        // -------------------------------------------------------------------------------- loader
        reg_dec<80>();
        const int w = warp - 8;
        typename S::Cursor at;
        at.set(p, pos, geo);
        // lane l holds key 32 w + l of a unit: its element offset, -1 to fill with zeros
        const auto lookup = [&]() -> int64_t {
            const int j = at.g.lo + at.at.c * KC + w * 32 + lane;
            if (j >= at.g.hi) return -1;
            const int64_t o = key_offset(p, at.at.r, j);
            return o < 0 ? -1 : o + (int64_t)(at.at.h * p.head_stride);
        };
        // 32 rows of a tile by this warp
        const auto copy_rows = [&](uint32_t tile, int row0, const void *base, int64_t off) {
#pragma unroll 4
            for (int i = 0; i < PIECES; ++i) {
                const int lr = i * ROWS_PER + lane / PIECES, c = lane % PIECES, row = row0 + lr;
                const int64_t o = __shfl_sync(0xffffffffu, off, lr);
                const bool live = o >= 0 && c * 8 < (int)p.head_dim;
                cp16(tile + (c >> 3) * (F::TILE / F::HALVES) + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                     static_cast<const uint16_t *>(base) + (live ? o + c * 8 : 0), live);
            }
        };
        // copies not yet handed over, oldest first: at most two groups stay in flight behind the newest
        uint64_t *pend[3] = {nullptr, nullptr, nullptr};
        int npend = 0;
        uint32_t clean[3] = {0, 0, 0};  // a V tile to clear of infinities and NaNs first: its address, else 0
        uint32_t clean_item[3] = {0, 0, 0};
        const auto hand_over = [&]() {  // the oldest: its copies have landed
            if (clean[0]) {
                bool bad = false;
                for (int i = 0; i < PIECES; ++i) {
                    const int row = w * 32 + i * ROWS_PER + lane / PIECES, c = lane % PIECES;
                    const uint32_t a = clean[0] - sbase + (c >> 3) * (F::TILE / F::HALVES) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                    uint4 *v = reinterpret_cast<uint4 *>(smem + a);
                    uint4 x = *v;
                    bool b = false;
                    x.x = finite2<TYPE>(x.x, b);
                    x.y = finite2<TYPE>(x.y, b);
                    x.z = finite2<TYPE>(x.z, b);
                    x.w = finite2<TYPE>(x.w, b);
                    if (b) *v = x;
                    bad |= b;
                }
                if (bad) poison[(clean_item[0] - 1) & 7] = clean_item[0];
            }
            fence_proxy_async_smem();
            mbar_arrive(pend[0]);
            pend[0] = pend[1];
            pend[1] = pend[2];
            clean[0] = clean[1];
            clean[1] = clean[2];
            clean_item[0] = clean_item[1];
            clean_item[1] = clean_item[2];
            --npend;
        };
        const auto push = [&](uint64_t *b, uint32_t tile_to_clean, uint32_t item) {
            cp_commit();
            pend[npend] = b;
            clean[npend] = tile_to_clean;
            clean_item[npend] = item;
            ++npend;
            if (npend == 3) {
                cp_wait<2>();
                hand_over();
            }
        };
        const auto drain = [&]() {
            cp_wait<0>();
            while (npend) hand_over();
        };
        // waits until a buffer is free; everything loaded is handed over before it blocks
        const auto room = [&](uint64_t *b, uint32_t parity) -> bool {
            if (__all_sync(0xffffffffu, mbar_test_wait(b, parity))) return true;
            drain();
            const bool ok = mbar_wait_bounded(b, parity, p.err, 30);
            return __all_sync(0xffffffffu, ok);
        };
        uint32_t e = 0, item = 0;
        int64_t off = lookup();
        bool fresh = true, ok = true;
        int all_lo = 0, all_hi = 0;
        for (int i = 0; i < n && ok; ++i) {
            const int64_t cur = off;
            const Pos here = at.at;
            const Req q = at.q;
            const int j0 = at.g.lo + at.at.c * KC;
            const bool ends = at.item_end();
            if (fresh) item_limits(p, q, here.t, all_lo, all_hi);
            const bool partial = j0 < all_lo || j0 + KC > all_hi;
            if (i + 1 < n) {
                at.next(p);
                off = lookup();
            }
            // K
            uint32_t st = e % NS, tile = sbase + F::RING_OFF + st * F::TILE;
            ok = room(&bar->empty[st], ((e / NS) & 1) ^ 1);
            if (!ok) break;
            copy_rows(tile, w * 32, p.k, cur);
            push(&bar->full[st], 0, 0);
            ++e;
            if (fresh) {  // the item's query rows
                ok = room(&bar->q_empty, (item & 1) ^ 1);
                if (!ok) break;
                const int rows = q.nq * (int)p.gd.d;
                for (int b = 0; b < 2; ++b) {
                    const int lr = w * 64 + b * 32 + lane, row = here.t * TR + lr;
                    int64_t o = -1;
                    if (row < rows) {
                        const uint32_t tok = p.gd.div((uint32_t)row);
                        o = (int64_t)((uint64_t)(q.q0 + tok) * p.q_stride +
                                      (uint64_t)(here.h * p.gd.d + row - tok * p.gd.d) * p.head_dim);
                    }
                    // rows 0-127 and 128-255 are a tile each
                    copy_rows(sbase + F::Q_OFF + (w >> 1) * F::TILE, (w & 1) * 64 + b * 32, p.q, o);
                }
                push(&bar->q_full, 0, 0);
                fresh = false;
            }
            // V
            st = e % NS;
            tile = sbase + F::RING_OFF + st * F::TILE;
            ok = room(&bar->empty[st], ((e / NS) & 1) ^ 1);
            if (!ok) break;
            copy_rows(tile, w * 32, p.v, cur);
            push(&bar->full[st], partial ? tile : 0, item + 1);
            ++e;
            if (ends) {
                fresh = true;
                ++item;
            }
        }
        drain();
    } else if (wg == 3) {
        // ---------------------------------------------------------------------------- the products
        reg_dec<64>();
        if (warp == 12) {
            constexpr uint32_t id_s = idesc16(TYPE, 128, KC, 0), id_o = idesc16(TYPE, 128, DP, 1);
            constexpr uint32_t HALF = F::TILE / F::HALVES;
            typename S::Cursor at;
            at.set(p, pos, geo);
            const auto scores = [&](int t, uint32_t ktile) {
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        const uint32_t o = (k >> 2) * HALF + (k & 3) * 32;
                        umma_bf16(tmem + s_col(t), sdesc_k_sw128(sbase + F::Q_OFF + t * F::TILE + o),
                                  sdesc_k_sw128(ktile + o), id_s, k != 0);
                    }
                    umma_commit(&bar->s_full[t]);
                }
                __syncwarp();
            };
            const auto values = [&](int t, uint32_t vtile, bool first) {
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < KC / 16; ++k)
                        umma_bf16_ts(tmem + o_col(t), tmem + s_col(t) + k * 8, sdesc_n_sw128(vtile + k * 2048, HALF), id_o,
                                     !(first && k == 0));
                }
                __syncwarp();
            };
            const auto commit = [&](uint64_t *b) {
                if (elect_one()) umma_commit(b);
                __syncwarp();
            };
            const auto wait = [&](uint64_t *b, uint32_t parity, int code) -> bool {
                const bool ok = mbar_wait_bounded(b, parity, p.err, code);
                const bool all = __all_sync(0xffffffffu, ok);
                tc_fence_after();
                return all;
            };
            const auto tile = [&](uint32_t e) { return sbase + F::RING_OFF + (e % NS) * F::TILE; };
            // entries of the ring: unit i's K is 2 i, its V 2 i + 1
            uint32_t item = 0, handed[2] = {0, 0};  // P tiles taken from each softmax warpgroup
            int nh = halves(p, at.q, at.at.t);
            const auto unit_scores = [&](int t, int i) {  // S_t of unit i (the cursor's)
                const uint32_t ek = 2 * i;
                scores(t, tile(ek));
                if (t == nh - 1) {
                    commit(&bar->empty[ek % NS]);
                    if (at.item_end() || i == n - 1) commit(&bar->q_empty);
                }
            };
            bool ok = wait(&bar->q_full, 0, 31) && wait(&bar->full[0], 0, 32);
            for (int t = 0; t < nh && ok; ++t) unit_scores(t, 0);
            bool first = true;
            for (int i = 0; i < n && ok; ++i) {
                const bool last = at.item_end() || i == n - 1;  // the item's last unit in this CTA
                const uint32_t ev = 2 * i + 1, ek = 2 * i + 2;
                ok = wait(&bar->full[ev % NS], (ev / NS) & 1, 33);
                for (int t = 0; t < nh && ok; ++t) {
                    ok = wait(&bar->p_full[t], handed[t] & 1, 34);
                    if (!ok) break;
                    ++handed[t];
                    values(t, tile(ev), first);
                    if (last) commit(&bar->o_full[t]);
                    if (t == nh - 1) commit(&bar->empty[ev % NS]);
                    if (!last) {
                        if (t == 0) {
                            ok = wait(&bar->full[ek % NS], (ek / NS) & 1, 35);
                            if (!ok) break;
                            at.next(p);
                        }
                        unit_scores(t, i + 1);
                    }
                }
                first = last;
                if (ok && last && i + 1 < n) {
                    ++item;
                    at.next(p);
                    nh = halves(p, at.q, at.at.t);
                    ok = wait(&bar->q_full, item & 1, 36) && wait(&bar->full[ek % NS], (ek / NS) & 1, 37);
                    for (int t = 0; t < nh && ok; ++t) unit_scores(t, i + 1);
                }
            }
            // every product has completed before tensor memory is freed, also after a wait gave up
            commit(&bar->done);
            mbar_wait_bounded(&bar->done, 0, nullptr, 0);
        }
    } else {
        // -------------------------------------------------------------------------------- softmax
        reg_inc<184>();
        const int t = wg, r = threadIdx.x & 127;  // tile of the item, row of the tile
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes: lane number << 16
        const uint32_t s_at = tmem + s_col(t) + lanes, o_at = tmem + o_col(t) + lanes;
        typename S::Cursor at;
        at.set(p, pos, geo);
        uint32_t item = 0, taken = 0, joined = 0;  // items met; score tiles and outputs taken
        int segment = 0, first_c = 0;
        bool fresh = true, ok = true;
        float m = -INFINITY, l = 0.0f;
        int lo = 0, hi = 0, all_lo = 0, all_hi = 0;
        for (int i = 0; i < n; ++i) {
            const int rows = at.q.nq * (int)p.gd.d, row0 = at.at.t * TR + t * 128;
            if (row0 >= rows) {  // no rows in this half: its products are not issued
                if (at.item_end()) {
                    ++segment;
                    ++item;
                }
                if (i + 1 < n) at.next(p);
                continue;
            }
            if (fresh) {
                first_c = at.at.c;
                m = -INFINITY;
                l = 0.0f;
                int dummy;
                row_limits(p, at.q, min(row0 + r, rows - 1), lo, hi);
                row_limits(p, at.q, row0, dummy, all_hi);
                row_limits(p, at.q, min(row0 + 128, rows) - 1, all_lo, dummy);
            }
            ok = mbar_wait_bounded(&bar->s_full[t], taken & 1, p.err, 38);
            if (!__all_sync(0xffffffffu, ok)) break;
            ++taken;
            tc_fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(s_at + c * 32, s[c]);
            tmem_ld_wait();
            const int j0 = at.g.lo + at.at.c * KC;
            if (j0 < all_lo || j0 + KC > all_hi) {
                const int a = lo - j0, b = hi - j0;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (c * 32 + x < a || c * 32 + x >= b) s[c][x] = 0xFF800000u;  // -infinity
            }
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
                for (int x = 1; x < 32; ++x) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][x]));
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
            if (fresh) {
                m = top;
            } else {
                const bool grow = top > m + GROW || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, grow)) {
                    // S_t(i) completed, so PV_t(i - 1) has too: O is at rest until P_t(i) is handed over
                    const float mn = grow ? top : m;
                    const float al = grow ? ex2(m - mn) : 1.0f;
                    m = mn;
                    l *= al;
#pragma unroll 1
                    for (int c = 0; c < DP / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(o_at + c * 32, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * al);
                        tmem_st32(o_at + c * 32, o);
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), rf2 = make_float2(-ref, -ref);
            float2 sum[2] = {make_float2(0, 0), make_float2(0, 0)};
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                uint32_t pk[32];
#pragma unroll
                for (int x = 0; x < 32; ++x) {
                    const int c = hh * 2 + x / 16, y = (x % 16) * 2;
                    float2 v = make_float2(__uint_as_float(s[c][y]), __uint_as_float(s[c][y + 1]));
                    v = __ffma2_rn(v, sc2, rf2);
                    v.x = ex2(v.x);
                    v.y = ex2(v.y);
                    sum[x & 1] = __fadd2_rn(sum[x & 1], v);
                    pk[x] = pack2(TYPE, v.x, v.y);
                }
                tmem_st32(s_at + hh * 32, pk);
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&bar->p_full[t]);
            fresh = false;
            if (at.item_end() || i == n - 1) {
                ok = mbar_wait_bounded(&bar->o_full[t], joined & 1, p.err, 39);
                if (!__all_sync(0xffffffffu, ok)) break;
                ++joined;
                tc_fence_after();
                const bool whole = first_c == 0 && at.item_end();
                const size_t slot = (size_t)blockIdx.x * 2 + (segment ? 1 : 0);
                const int row = row0 + r;
                const bool live = row < rows;
                const bool cleaned = poison[item & 7] == item + 1;
                const bool some = l > 0.0f || l != l;
                const float inv = whole ? (some ? 1.0f / l : 0.0f) : 1.0f;
                const uint32_t tok = p.gd.div((uint32_t)(live ? row : 0));
                const uint32_t head = at.at.h * p.gd.d + ((live ? row : 0) - tok * p.gd.d);
                const uint64_t oe = (uint64_t)(at.q.q0 + tok) * p.out_stride + (uint64_t)head * p.head_dim;
                float *po = p.part_o + (slot * TR + t * 128 + r) * DP;
#pragma unroll 1
                for (int c = 0; c < DP / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(o_at + c * 32, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int d = c * 32 + g * 8;
                        if (!live || d >= (int)p.head_dim) continue;
                        float v[8];
#pragma unroll
                        for (int x = 0; x < 8; ++x) v[x] = __uint_as_float(o[g * 8 + x]) * inv;
                        if (cleaned) {
                            int il, ih;
                            item_limits(p, at.q, at.at.t, il, ih);
                            const int s0 = at.g.lo + first_c * KC, s1 = min(at.g.lo + (at.at.c + 1) * KC, at.g.hi);
                            for (int j = s0; j < s1; j += KC)
                                if (j < il || j + KC > ih)
                                    for (int x = 0; x < 8; ++x)
                                        v[x] += nonfinite_v(p, at.at.r, at.at.h, d + x, j, min(j + KC, s1), lo, hi);
                        }
                        if (whole) store8(p.out, oe + d, TYPE, v);
                        else store8(po, d, T_F32, v);
                    }
                    __syncwarp();
                }
                if (live) {
                    if (!whole) {
                        float *pm = p.part_ml + (slot * TR + t * 128 + r) * 2;
                        pm[0] = m;
                        pm[1] = l;
                    } else if (p.lse) {
                        p.lse[(uint64_t)(at.q.q0 + tok) * (p.n_kv * p.gd.d) + head] =
                            some ? (m + log2f(l)) * LN2 : -INFINITY;
                    }
                }
                tc_fence_before();
                ++segment;
                ++item;
                fresh = true;
            }
            if (i + 1 < n) at.next(p);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int TYPE, int DP>
int launch(AttnParams p, cudaStream_t s) {
    using F = Chunk<DP>;
    static unsigned long long done = 0;
    if (attr_pending(done)) {
        cudaError_t e = cudaFuncSetAttribute(k_attn_chunk<TYPE, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
        if (e != cudaSuccess) return (int)e;
        attr_mark(done);
    }
    const uint32_t grid = SMS;
    p.part_ml = p.part_o + (size_t)grid * 2 * TR * DP;
    cudaError_t e = launch_pdl(k_attn_chunk<TYPE, DP>, dim3(grid), dim3(NTHREADS), F::SMEM, s, p);
    if (e == cudaSuccess) e = launch_pdl(k_attn_join<S, TR, DP>, dim3(grid - 1, 8), dim3(128), 0, s, p, (int)grid);
    return (int)e;
}

}  // namespace
}  // namespace attn

size_t attn_chunk_workspace_bytes(uint32_t head_dim) {
    const size_t dp = head_dim <= 64 ? 64 : 128;
    return head_dim > 128 ? 0 : SMS * 2 * attn::TR * (dp + 2) * 4;
}
int launch_attn_chunk(const AttnParams &p, cudaStream_t s) {
    if (!attn_chunk_ok_types(p.io_type, p.cache_type, p.head_dim)) return CK_ERR_SHAPE;
    if (p.cache_type == T_BF16)
        return p.head_dim <= 64 ? attn::launch<T_BF16, 64>(p, s) : attn::launch<T_BF16, 128>(p, s);
    return p.head_dim <= 64 ? attn::launch<T_F16, 64>(p, s) : attn::launch<T_F16, 128>(p, s);
}

}  // namespace ck
