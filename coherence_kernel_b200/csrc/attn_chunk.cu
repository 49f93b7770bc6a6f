// attn_chunk.cu -- attention of many rows (long chunks of new tokens, or many heads over one K/V head) over
// the paged cache, on the fifth-generation tensor cores.
//
// The same one-pass softmax as attn_paged.cu with tiles of 256 rows and units of 128 keys.  One CTA per
// SM of four warpgroups:
//   0, 1  softmax: each owns 128 rows, a thread one row.  Reads its scores from tensor memory (all 128 of
//         a unit in registers), masks, keeps maximum and sum, and writes P as bf16 / f16 pairs over the
//         scores it came from -- the A operand of the second product never leaves tensor memory.  P is handed over
//         in two halves, so that the product over the first runs beside the second's exponentials
//   2     loader: one warp issues TMA loads of K and V (a box of up to 64 tokens of a page, its page looked up by a
//         lane a unit ahead) and of the queries into a ring of four 128-key tiles, 128-byte swizzle; the others clean
//         V tiles on the edge of the mask.  Pages that hold no multiple of 8 tokens, and query groups that
//         are no power of two, come by 16-byte asynchronous copies instead
//   3     one warp issues the products: S_t = Q_t K^T (both operands in shared memory) and
//         O_t += P_t V (P in tensor memory, V as an N-major B operand straight from its row layout)
// Tensor memory: S_0 S_1 O_0 O_1, 128 columns each.  The issue order PV_0(i) S_0(i+1) PV_1(i) S_1(i+1) keeps the
// tensor core on one half while the other half's softmax runs; S_t(i+1) may follow PV_t(i) unwaited, since
// one thread's products execute in order.
//
// O is rescaled only when a row's maximum has grown by more than 8 (in log2 units) since the maximum
// its weights refer to: weights stay below 2^8, exactly representable scaling, and most units skip the
// round trip of O through registers.  P is rounded once to the cache's type, half an ulp of each weight:
// against 64 bits the outputs are off by 1.4 times what their own rounding alone gives (2048 new tokens of 8192, bf16:
// 0.0023 of their norm for 0.0017).  Scores, sums and O are fp32.  f16 weights are taken times 2^13 and rescaled at a
// growth of 2.9, which keeps them below 2^15.9, within f16: only those under 2^-27 of their row's largest fall among f16's
// subnormals, where a weight is off by at most 2^-38 of the largest.  The maximum they refer to is rounded down to a whole
// number, so that neither the shift nor taking it back rounds anything (2048 new tokens of 8192: 247 us, as in bf16).
//
// Bounds per unit: the tensor core (4 x 128 x 128 x 128 multiply-adds, 2048 cycles), the exponentials (2 x 128 x 128 at 16
// per cycle, 2048 cycles) and the tiles' way from L2 (64 KB at about 26 bytes per cycle, 2500 cycles) are close to
// each other, and the chain scores - softmax - product of a half leaves gaps between them: about 4100 cycles.
// 2048 new tokens of 8192, 32 heads over 8 of 128: 241 to 249 us, 980 TFLOP/s, 60% of the measured bf16 GEMM rate (tensor pipe 47%
// active, special-function unit 47%).  Tried and slower: steps of 64 keys with their own score columns (271 us: an
// N = 64 product of two shared-memory operands waits for shared memory), two threads per row (253), a
// polynomial for a share of the exponentials (262 to 349, the share from 1/8 to 1/2).
#include "attn_sched.cuh"

namespace ck {
namespace attn {
namespace {

constexpr int TR = 256, KC = 128;
using S = Sched<TR, KC, true>;
constexpr int NTHREADS = 512;

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
    uint64_t full[4], empty[4], raw[4], q_full, q_empty, s_full[2], p_half[2], p_full[2], o_full[2], done;
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

CK_DEV float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// queries: a 3D map (dim, head, token), a box of 64 dims of a group's heads for 128 / group tokens: 128 rows in tile order
CK_DEV void tma_load_q(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int d, int head, int tok) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(d), "r"(head), "r"(tok)
        : "memory");
}
inline int make_q_map(CUtensorMap *m, const AttnParams &p, int tokens) {
    const cuuint64_t dims[3] = {p.head_dim, (cuuint64_t)p.n_kv * p.gd.d, p.ntok};
    const cuuint64_t strides[2] = {p.head_dim * 2ull, p.q_stride * 2};
    const cuuint32_t box[3] = {64, p.gd.d, (cuuint32_t)tokens};
    return encode_map(m, p.q, p.cache_type, 3, dims, strides, box);
}

template <int TYPE, int DP, bool TMA>
__global__ void __launch_bounds__(NTHREADS, 1)
    k_attn_chunk(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap, int box, int qbox) {
    using F = Chunk<DP>;
    constexpr int PIECES = DP / 8;           // 16-byte pieces of a row
    constexpr int ROWS_PER = 32 / PIECES;    // rows one warp instruction copies
    constexpr int NS = F::STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ typename S::Shared sh;
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t item_info[8];  // by item modulo 8: its units in this CTA, 1 << 30 if it is the last, 1 << 31 if both
                                       // halves hold rows
    __shared__ uint32_t poison[8];  // item number + 1 of an item whose V was cleaned, by item modulo 8
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    Bars *bar = reinterpret_cast<Bars *>(smem + F::BAR_OFF);
    const uint32_t sbase = smem_u32(smem);
    const int wg = threadIdx.x >> 7, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_trigger_small();
    if (TMA && threadIdx.x == 0) {
        prefetch_tmap(&kmap);
        prefetch_tmap(&vmap);
        if (qbox) prefetch_tmap(&qmap);
    }
    grid_dep_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.err = 0;
    long long U;
    int C;
    Pos pos;
    Geo geo;
    const bool part = S::find(p, sh, (int)gridDim.x, (int)blockIdx.x, U, C, pos, geo);
    S::leave_cut(p, U, C, pos, geo);
    if (!part) return;
    const int n = (int)(S::start(U, C, blockIdx.x + 1) - S::start(U, C, blockIdx.x));
    if (pos.c >= geo.nch && n <= geo.nch + S::EXTRA - pos.c) return;  // no unit with keys
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&bar->full[i], TMA ? 1 : 128);
            mbar_init(&bar->empty[i], 1);
            mbar_init(&bar->raw[i], 1);
        }
        mbar_init(&bar->q_full, qbox ? 1 : (TMA ? 96 : 128) + 1);
        mbar_init(&bar->q_empty, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&bar->s_full[t], 1);
            mbar_init(&bar->p_half[t], 128);
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
        reg_dec<72>();
        const int w = warp - 8;
        constexpr uint32_t HALF = F::TILE / F::HALVES;
        typename S::Items it;
        it.set(p, sh, n);
        const auto room = [&](uint64_t *b, uint32_t parity) -> bool {
            return __all_sync(0xffffffffu, mbar_wait_short(b, parity, p.err, 30));
        };
        // 32 rows of a tile by one warp: lane l has the element offset of row l, -1 to fill it with zeros
        const auto copy_rows = [&](uint32_t tile, int row0, const void *base, int64_t off) {
#pragma unroll 4
            for (int i = 0; i < PIECES; ++i) {
                const int lr = i * ROWS_PER + lane / PIECES, c = lane % PIECES, row = row0 + lr;
                const int64_t o = __shfl_sync(0xffffffffu, off, lr);
                const bool live = o >= 0 && c * 8 < (int)p.head_dim;
                cp16(tile + (c >> 3) * HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                     static_cast<const uint16_t *>(base) + (live ? o + c * 8 : 0), live);
            }
        };
        // The copies arrive on the barrier themselves once they have landed, so the loader runs as far ahead as
        // the ring lets it; the thread that issues the products runs the proxy fence after its wait.
        const auto hand_over = [&](uint64_t *b) {
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
        };
        // query rows 32 b .. 32 b + 31 of the item; rows 0-127 and 128-255 are a tile each
        const auto copy_queries = [&](int b) {
            const int row = it.at.t * TR + b * 32 + lane;
            int64_t o = -1;
            if (row < it.q.nq * (int)p.gd.d) {
                const uint32_t tok = p.gd.div((uint32_t)row);
                o = (int64_t)((uint64_t)(it.q.q0 + tok) * p.q_stride +
                              (uint64_t)(it.at.h * p.gd.d + row - tok * p.gd.d) * p.head_dim);
            }
            copy_rows(sbase + F::Q_OFF + (b >> 2) * F::TILE, (b & 3) * 32, p.q, o);
        };
        // The first rows of a V tile with keys that only some rows see, `step` threads together: infinities and NaNs
        // become zeros, and so do the rows of keys past the last (n_keys on), which hold whatever the page does.
        const auto clean = [&](uint32_t tile, uint32_t item, int rows, int first, int step, int n_keys) {
            bool bad = false;
            for (int i = first; i < rows * PIECES; i += step) {
                const int row = i / PIECES, c = i % PIECES;
                const uint32_t a = tile - sbase + (c >> 3) * HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                uint4 *v = reinterpret_cast<uint4 *>(smem + a);
                if (row >= n_keys) {
                    *v = make_uint4(0, 0, 0, 0);
                    continue;
                }
                uint4 x = *v;
                bool b = false;
                x.x = finite2<TYPE>(x.x, b);
                x.y = finite2<TYPE>(x.y, b);
                x.z = finite2<TYPE>(x.z, b);
                x.w = finite2<TYPE>(x.w, b);
                if (b) *v = x;
                bad |= b;
            }
            if (bad) poison[item & 7] = item + 1;
        };
        // what the products' warp needs of an item, before the arrival that lets it at the queries
        const auto describe = [&](uint32_t item) {
            // the last item: what is left ends with it
            const bool last = it.left <= it.g.nch + S::EXTRA - it.c0;
            item_info[item & 7] = (uint32_t)(it.c1 - it.c0) | (uint32_t)last << 30 |
                                  (uint32_t)(halves(p, it.q, it.at.t) - 1) << 31;
        };
        uint32_t e = 0, item = 0;  // ring entries and items so far
        bool ok = true;
        if constexpr (TMA) {
            if (w == 0) {
                // K and V: a lane per box of the unit looks its page up a unit ahead and issues its loads
                const int boxes = KC / box;
                uint32_t to_raw = 0;  // a bit per stage: its last loads went to the raw barrier
                uint32_t raw_phase = 0;
                const auto lookup = [&](int c) -> int2 {  // page (past the last: zeros) and token of the lane's box
                    const int j = it.g.lo + c * KC + lane * box;
                    if (lane >= boxes || j >= it.g.hi) return make_int2((int)p.n_blocks, 0);
                    const uint32_t b = p.btd.div((uint32_t)j);
                    const int pg = p.table[(uint64_t)it.at.r * p.table_stride + b];
                    return make_int2(pg >= 0 && pg < (int)p.n_blocks ? pg : (int)p.n_blocks, j - (int)(b * p.btd.d));
                };
                do {
                    int all_lo, all_hi;
                    item_limits(p, it.q, it.at.t, all_lo, all_hi);
                    int2 next = lookup(it.c0);
                    for (int c = it.c0; c < it.c1 && ok; ++c) {
                        const int2 at = next;
                        if (c + 1 < it.c1) next = lookup(c + 1);
                        const int j0 = it.g.lo + c * KC;
                        const bool partial = j0 < all_lo || j0 + KC > all_hi;
                        for (int kv = 0; kv < 2; ++kv, ++e) {
                            const uint32_t st = e % NS, tile = sbase + F::RING_OFF + st * F::TILE + lane * box * 128;
                            ok = room(&bar->empty[st], ((e / NS) & 1) ^ 1);
                            if (!ok) break;
                            const bool raw = kv && partial;
                            uint64_t *full = raw ? &bar->raw[st] : &bar->full[st];
                            to_raw = (to_raw & ~(1u << st)) | (uint32_t)raw << st;
                            raw_phase ^= (uint32_t)raw << st;  // after it: the parity of the next use
                            if (lane == 0) mbar_arrive_expect_tx(full, F::TILE);
                            __syncwarp();
                            if (lane < boxes) {
                                const CUtensorMap *map = kv ? &vmap : &kmap;
#pragma unroll
                                for (int x = 0; x < F::HALVES; ++x)
                                    tma_load_kv(tile + x * HALF, map, full, x * 64, it.at.h, at.y, at.x);
                            }
                            __syncwarp();
                            if (qbox && kv == 0 && c == it.c0) {
                                ok = room(&bar->q_empty, (item & 1) ^ 1);
                                if (!ok) break;
                                if (lane == 0) {
                                    describe(item);
                                    const int nh = halves(p, it.q, it.at.t), tok = it.q.q0 + (it.at.t * 2) * qbox;
                                    mbar_arrive_expect_tx(&bar->q_full, nh * F::TILE);
                                    for (int t = 0; t < nh; ++t)
                                        for (int x = 0; x < F::HALVES; ++x)
                                            tma_load_q(sbase + F::Q_OFF + t * F::TILE + x * HALF, &qmap, &bar->q_full,
                                                       x * 64, it.at.h * p.gd.d, tok + t * qbox);
                                }
                                __syncwarp();
                            }
                        }
                    }
                    ++item;
                } while (ok && it.next(p));
                // after a wait gave up, no load outlives the block
                for (uint32_t x = e > NS ? e - NS : 0; !ok && x < e; ++x) {
                    const uint32_t st = x % NS;
                    if (to_raw >> st & 1) mbar_wait_short(&bar->raw[st], (raw_phase >> st & 1) ^ 1, nullptr, 0);
                    else mbar_wait_short(&bar->full[st], (x / NS) & 1, nullptr, 0);
                }
            } else {
                // the queries, and the V tiles to clean
                const int me = threadIdx.x - 288;  // 0 .. 95
                uint32_t raw_parity = 0;           // a bit per stage
                // the three warps go on or give up together: they meet at a barrier below
                const auto together = [](bool ok) -> bool {
                    uint32_t r;
                    asm volatile(
                        "{\n .reg .pred a, b;\n setp.ne.u32 a, %1, 0;\n barrier.cta.red.and.pred b, 2, 96, a;\n selp.u32 %0, 1, 0, b;\n}"
                        : "=r"(r)
                        : "r"((uint32_t)ok)
                        : "memory");
                    return r != 0;
                };
                do {
                    if (!qbox) {
                        ok = together(mbar_wait_short(&bar->q_empty, (item & 1) ^ 1, p.err, 30));
                        if (!ok) break;
                        for (int b = w - 1; b < TR / 32; b += 3) copy_queries(b);
                        hand_over(&bar->q_full);
                        if (me == 0) {
                            describe(item);
                            mbar_arrive(&bar->q_full);
                        }
                    }
                    int all_lo, all_hi;
                    item_limits(p, it.q, it.at.t, all_lo, all_hi);
                    for (int c = it.c0; c < it.c1 && ok; ++c, e += 2) {
                        const int j0 = it.g.lo + c * KC;
                        if (j0 >= all_lo && j0 + KC <= all_hi) continue;
                        const uint32_t st = (e + 1) % NS;
                        ok = together(mbar_wait_short(&bar->raw[st], raw_parity >> st & 1, p.err, 41));
                        if (!ok) break;
                        raw_parity ^= 1u << st;
                        clean(sbase + F::RING_OFF + st * F::TILE, item, KC, me, 96, it.g.hi - j0);
                        fence_proxy_async_smem();
                        asm volatile("bar.sync 1, 96;" ::: "memory");
                        if (me == 0) mbar_arrive(&bar->full[st]);
                    }
                    ++item;
                } while (ok && it.next(p));
            }
        } else {
            // pages of other sizes: 16-byte copies, lane l of warp w looks up key 32 w + l a unit ahead
            const auto lookup = [&](int c) -> int64_t {
                const int j = it.g.lo + c * KC + w * 32 + lane;
                if (j >= it.g.hi) return -1;
                const int64_t o = key_offset(p, it.at.r, j);
                return o < 0 ? -1 : o + (int64_t)(it.at.h * p.head_stride);
            };
            do {
                int all_lo, all_hi;
                item_limits(p, it.q, it.at.t, all_lo, all_hi);
                int64_t next = lookup(it.c0);
                for (int c = it.c0; c < it.c1 && ok; ++c) {
                    const int64_t off = next;
                    if (c + 1 < it.c1) next = lookup(c + 1);
                    const int j0 = it.g.lo + c * KC;
                    const bool partial = j0 < all_lo || j0 + KC > all_hi;
                    for (int kv = 0; kv < 2; ++kv, ++e) {
                        const uint32_t st = e % NS, tile = sbase + F::RING_OFF + st * F::TILE;
                        ok = room(&bar->empty[st], ((e / NS) & 1) ^ 1);
                        if (!ok) break;
                        copy_rows(tile, w * 32, kv ? p.v : p.k, off);
                        if (kv && partial) {
                            cp_commit();
                            cp_wait<0>();
                            __syncwarp();  // a warp cleans the rows it copied
                            clean(tile + w * 32 * 128, item, 32, lane, 32, 32);
                            // ordinary stores: the copies' own arrival does not order them
                            fence_proxy_async_smem();
                            mbar_arrive(&bar->full[st]);
                        } else {
                            hand_over(&bar->full[st]);
                        }
                        if (kv == 0 && c == it.c0) {  // the item's queries
                            ok = room(&bar->q_empty, (item & 1) ^ 1);
                            if (!ok) break;
                            copy_queries(2 * w);
                            copy_queries(2 * w + 1);
                            hand_over(&bar->q_full);
                            if (threadIdx.x == 256) {
                                describe(item);
                                mbar_arrive(&bar->q_full);
                            }
                        }
                    }
                }
                ++item;
            } while (ok && it.next(p));
        }
        cp_commit();
        cp_wait<0>();  // no copy outlives the thread, also after a wait gave up
    } else if (wg == 3) {
        // ---------------------------------------------------------------------------- the products
        reg_dec<72>();
        if (warp == 12) {
            constexpr uint32_t id_s = idesc16(TYPE, 128, KC, 0), id_o = idesc16(TYPE, 128, DP, 1);
            constexpr uint32_t HALF = F::TILE / F::HALVES;
            const uint64_t q_desc = sdesc_k_sw128(sbase + F::Q_OFF), k_desc = sdesc_k_sw128(sbase + F::RING_OFF),
                           v_desc = sdesc_n_sw128(sbase + F::RING_OFF, HALF);
            constexpr uint32_t STAGE16 = F::TILE >> 4;  // descriptors count 16 bytes
            const auto commit = [&](uint64_t *b) {
                if (elect_one()) umma_commit(b);
                __syncwarp();
            };
            const auto wait = [&](uint64_t *b, uint32_t parity, int code) -> bool {
                const bool ok = mbar_wait_short(b, parity, p.err, code);
                return __all_sync(0xffffffffu, ok);
            };
            const auto wait_tile = [&](uint64_t *b, uint32_t parity, int code) -> bool {
                const bool ok = wait(b, parity, code);
                fence_proxy_async_smem();  // the loader's writes, before the tensor core reads them
                return ok;
            };
            const auto wait_weights = [&](uint64_t *b, uint32_t parity, int code) -> bool {
                const bool ok = wait(b, parity, code);
                tc_fence_after();
                return ok;
            };
            // S_t = Q_t K^T from ring stage st; free: barriers of what this was the last use of
            const auto scores = [&](int t, uint32_t st, bool k_done, bool q_done) {
                const uint64_t qd = q_desc + t * STAGE16, kd = k_desc + st * STAGE16;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        const uint32_t o = (k >> 2) * (HALF >> 4) + (k & 3) * 2;
                        umma_bf16(tmem + s_col(t), qd + o, kd + o, id_s, k != 0);
                    }
                    umma_commit(&bar->s_full[t]);
                    if (k_done) umma_commit(&bar->empty[st]);
                    if (q_done) umma_commit(&bar->q_empty);
                }
                __syncwarp();
            };
            // O_t (+)= P_t V over half h of the unit's keys, from ring stage st
            const auto values = [&](int t, int h, uint32_t st, bool first, bool v_done, bool o_done) {
                const uint64_t vd = v_desc + st * STAGE16;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < KC / 32; ++k) {
                        const int kk = h * (KC / 32) + k;
                        umma_bf16_ts(tmem + o_col(t), tmem + s_col(t) + kk * 8, vd + kk * 128, id_o, !(first && kk == 0));
                    }
                    if (v_done) umma_commit(&bar->empty[st]);
                    if (o_done) umma_commit(&bar->o_full[t]);
                }
                __syncwarp();
            };
            uint32_t e = 0, item = 0, handed[2] = {0, 0};  // ring entries, items, P tiles taken from each half
            bool ok = true;
            for (bool more = true; more && ok;) {
                ok = wait_tile(&bar->q_full, item & 1, 31) && wait_tile(&bar->full[e % NS], (e / NS) & 1, 32);
                if (!ok) break;
                const uint32_t info = item_info[item & 7];
                const int nh = 1 + (int)(info >> 31), units = (int)(info & 0x3fffffffu);
                more = !(info >> 30 & 1);
                for (int t = 0; t < nh; ++t) scores(t, e % NS, t == nh - 1, t == nh - 1 && units == 1);
                ++e;
                for (int c = 0; c < units && ok; ++c) {
                    const bool last = c == units - 1;
                    const uint32_t sv = e % NS, sk = (e + 1) % NS;
                    ok = wait_tile(&bar->full[sv], (e / NS) & 1, 33);
                    for (int t = 0; t < nh && ok; ++t) {
                        ok = wait_weights(&bar->p_half[t], handed[t] & 1, 34);
                        if (!ok) break;
                        values(t, 0, sv, c == 0, false, false);
                        ok = wait_weights(&bar->p_full[t], handed[t] & 1, 36);
                        if (!ok) break;
                        ++handed[t];
                        values(t, 1, sv, c == 0, t == nh - 1, last);
                        if (!last) {
                            if (t == 0) ok = wait_tile(&bar->full[sk], ((e + 1) / NS) & 1, 35);
                            if (ok) scores(t, sk, t == nh - 1, t == nh - 1 && c == units - 2);
                        }
                    }
                    e += last ? 1 : 2;
                }
                ++item;
            }
            // every product has completed before tensor memory is freed, also after a wait gave up
            commit(&bar->done);
            mbar_wait_short(&bar->done, 0, nullptr, 0);
        }
    } else {
        // -------------------------------------------------------------------------------- softmax
        reg_inc<184>();
        // log2 growth of a row's maximum that makes O rescale, and the power of two that weights are raised by
        constexpr float GROW = TYPE == T_F16 ? 2.9f : 8.0f, LIFT = TYPE == T_F16 ? 13.0f : 0.0f;
        constexpr float DOWN = TYPE == T_F16 ? 0x1p-13f : 1.0f;
        const int t = wg, r = threadIdx.x & 127;  // tile of the item, row of the tile
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes: lane number << 16
        const uint32_t s_at = tmem + s_col(t) + lanes, o_at = tmem + o_col(t) + lanes;
        typename S::Items it;
        it.set(p, sh, n);
        uint32_t taken = 0, joined = 0;  // score tiles and outputs taken
        uint32_t item = 0;
        int segment = 0;
        bool ok = true;
        do {
            const int rows = it.q.nq * (int)p.gd.d, row0 = it.at.t * TR + t * 128;
            const size_t slot = (size_t)blockIdx.x * 2 + (segment ? 1 : 0);
            ++segment;
            ++item;
            if (row0 >= rows) continue;  // no rows in this half: its products are not issued
            int lo, hi, all_lo, all_hi;
            float m = -INFINITY, l = 0.0f;
            {
                int dummy;
                row_limits(p, it.q, min(row0 + r, rows - 1), lo, hi);
                row_limits(p, it.q, row0, dummy, all_hi);
                row_limits(p, it.q, min(row0 + 128, rows) - 1, all_lo, dummy);
            }
            int j0 = it.g.lo + it.c0 * KC;
            for (int c = it.c0; c < it.c1; ++c, j0 += KC) {
                ok = mbar_wait_short(&bar->s_full[t], taken & 1, p.err, 38);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ++taken;
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int b = 0; b < 4; ++b) tmem_ld32(s_at + b * 32, s[b]);
                tmem_ld_wait();
                if (j0 < all_lo || j0 + KC > all_hi) {
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        // bit x: the row sees key j0 + 32 b + x
                        const int a = min(max(lo - j0 - b * 32, 0), 32), z = min(max(hi - j0 - b * 32, 0), 32);
                        const uint32_t see = (uint32_t)((1ull << z) - 1) & ~(uint32_t)((1ull << a) - 1);
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (!(see & (1u << x))) s[b][x] = 0xFF800000u;  // -infinity
                    }
                }
                float mx[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    mx[b] = __uint_as_float(s[b][0]);
#pragma unroll
                    for (int x = 1; x + 1 < 32; x += 2) mx[b] = max3(mx[b], __uint_as_float(s[b][x]), __uint_as_float(s[b][x + 1]));
                }
                const float top = fmaxf(max3(max3(mx[0], __uint_as_float(s[0][31]), __uint_as_float(s[1][31])), mx[1],
                                             __uint_as_float(s[2][31])),
                                        max3(mx[2], mx[3], __uint_as_float(s[3][31]))) *
                                  p.scale_log2;
                const float whole_top = LIFT != 0.0f ? floorf(top) : top;
                if (c == it.c0) {
                    m = whole_top;
                } else {
                    const bool grow = top > m + GROW || (m == -INFINITY && top > m);
                    if (__any_sync(0xffffffffu, grow)) {
                        // S_t of this unit completed, so PV_t of the last one has too: O is at rest until P_t is
                        // handed over
                        const float mn = grow ? whole_top : m;
                        const float al = grow ? ex2(m - mn) : 1.0f;
                        m = mn;
                        l *= al;
#pragma unroll 1
                        for (int b = 0; b < DP / 16; ++b) {
                            uint32_t o[16];
                            tmem_ld16(o_at + b * 16, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * al);
                            tmem_st16(o_at + b * 16, o);
                        }
                    }
                }
                const float ref = (m == -INFINITY ? 0.0f : m) - LIFT;
                const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), rf2 = make_float2(-ref, -ref);
                float2 sum[2] = {make_float2(0, 0), make_float2(0, 0)};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t pk[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        float2 v = make_float2(__uint_as_float(s[b][2 * x]), __uint_as_float(s[b][2 * x + 1]));
                        v = __ffma2_rn(v, sc2, rf2);
                        v.x = ex2(v.x);
                        v.y = ex2(v.y);
                        sum[x & 1] = __fadd2_rn(sum[x & 1], v);
                        pk[x] = pack2(TYPE, v.x, v.y);
                    }
                    tmem_st16(s_at + b * 16, pk);
                    if (b == 1) {  // the first half of the keys: its product can start
                        tmem_st_wait();
                        tc_fence_before();
                        mbar_arrive(&bar->p_half[t]);
                    }
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bar->p_full[t]);
            }
            if (!ok) break;
            ok = mbar_wait_short(&bar->o_full[t], joined & 1, p.err, 39);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++joined;
            tc_fence_after();
            const bool whole = it.whole();
            const int row = row0 + r;
            const bool live = row < rows;
            l *= DOWN;
            const bool some = l > 0.0f || l != l;
            const float inv = whole ? (some ? DOWN / l : 0.0f) : DOWN;
            const uint32_t tok = p.gd.div((uint32_t)(live ? row : 0));
            const uint32_t head = it.at.h * p.gd.d + ((live ? row : 0) - tok * p.gd.d);
            const uint64_t oe = (uint64_t)(it.q.q0 + tok) * p.out_stride + (uint64_t)head * p.head_dim;
            // a part's column d of all rows is contiguous: a warp's store is one line
            float *po = p.part_o + slot * (TR * DP) + t * 128 + r;
            const bool cleaned = poison[(item - 1) & 7] == item;
#pragma unroll 1
            for (int b = 0; b < DP / 16; ++b) {
                uint32_t o[16];
                tmem_ld16(o_at + b * 16, o);
                tmem_ld_wait();
                float v[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) v[x] = __uint_as_float(o[x]) * inv;
                if (cleaned && live) {
                    int il, ih;
                    item_limits(p, it.q, it.at.t, il, ih);
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        v[x] += nonfinite_v(p, it.at.r, it.at.h, b * 16 + x, it.g.lo + it.c0 * KC,
                                            min(it.g.lo + it.c1 * KC, it.g.hi), KC, il, ih, lo, hi);
                }
                if (!whole) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) po[(b * 16 + x) * TR] = v[x];
                } else if (live) {
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                        if (b * 16 + g * 8 < (int)p.head_dim) {
                            const float w[8] = {v[g * 8], v[g * 8 + 1], v[g * 8 + 2], v[g * 8 + 3],
                                                v[g * 8 + 4], v[g * 8 + 5], v[g * 8 + 6], v[g * 8 + 7]};
                            store8(p.out, oe + b * 16 + g * 8, TYPE, w);
                        }
                }
                __syncwarp();
            }
            if (!whole) {
                float *pm = p.part_ml + slot * (TR * 2) + t * 128 + r;
                pm[0] = m;
                pm[TR] = l;
            } else if (live && p.lse) {
                p.lse[(uint64_t)(it.q.q0 + tok) * (p.n_kv * p.gd.d) + head] = some ? (m + log2f(l)) * LN2 : -INFINITY;
            }
            tc_fence_before();
        } while (it.next(p));
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

// Joins the parts of an item that spans CTAs: block (j, y) takes JOIN_COLS columns of all rows of the item whose first
// cut is boundary j + 1, a thread a row, so that reads of a part's columns are whole lines.  Sixteen columns: all
// blocks are resident at once (17 ragged requests 54.8 us; 8 columns 55.8, 32 columns 56.7).
constexpr int JOIN_COLS = 16;
template <int DP>
__global__ void __launch_bounds__(TR) k_attn_join_chunk(const __grid_constant__ AttnParams p) {
    grid_dep_trigger_small();
    grid_dep_wait();
    Cut jt;
    const int d = (int)blockIdx.y * JOIN_COLS;
    if (d >= (int)p.head_dim || !find_joint<S>(p, (int)blockIdx.x + 1, jt)) return;
    const Req q = load_req(p, jt.at.r);
    const int r = threadIdx.x, row = jt.at.t * TR + r;
    if (row >= q.nq * (int)p.gd.d) return;
    float mm = -INFINITY;
    for (int i = 0; i < jt.n; ++i) mm = fmaxf(mm, p.part_ml[jt.slot(i) * (TR * 2) + r]);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, o[JOIN_COLS] = {};
#pragma unroll 2
    for (int i = 0; i < jt.n; ++i) {
        const size_t at = jt.slot(i);
        const float w = ex2(p.part_ml[at * (TR * 2) + r] - ref);
        ll += w * p.part_ml[at * (TR * 2) + TR + r];
#pragma unroll
        for (int x = 0; x < JOIN_COLS; ++x) o[x] += w * p.part_o[at * (TR * DP) + (d + x) * TR + r];
    }
    const bool some = ll > 0.0f || ll != ll;
    const float inv = some ? 1.0f / ll : 0.0f;
    const uint32_t tok = p.gd.div((uint32_t)row);
    const uint32_t head = jt.at.h * p.gd.d + (row - tok * p.gd.d);
    const uint64_t oe = (uint64_t)(q.q0 + tok) * p.out_stride + (uint64_t)head * p.head_dim + d;
#pragma unroll
    for (int g = 0; g < JOIN_COLS; g += 8)
        if (d + g < (int)p.head_dim) {
            const float v[8] = {o[g] * inv, o[g + 1] * inv, o[g + 2] * inv, o[g + 3] * inv,
                                o[g + 4] * inv, o[g + 5] * inv, o[g + 6] * inv, o[g + 7] * inv};
            store8(p.out, oe + g, p.io_type, v);
        }
    if (p.lse && d == 0)
        p.lse[(uint64_t)(q.q0 + tok) * (p.n_kv * p.gd.d) + head] = some ? (mm + log2f(ll)) * LN2 : -INFINITY;
}

template <int TYPE, int DP, bool TMA>
int launch(AttnParams p, int box, cudaStream_t s) {
    using F = Chunk<DP>;
    static unsigned long long done = 0;
    if (attr_pending(done)) {
        cudaError_t e = cudaFuncSetAttribute(k_attn_chunk<TYPE, DP, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
        if (e != cudaSuccess) return (int)e;
        attr_mark(done);
    }
    const uint32_t grid = SMS;
    p.part_ml = p.part_o + (size_t)grid * 2 * TR * DP;
    CUtensorMap kmap = {}, vmap = {}, qmap = {};
    // queries by TMA too where a 128-row tile is whole tokens of the group's heads (powers of two up to 128)
    const uint32_t group = p.gd.d;
    int qbox = TMA && group <= 128 && (group & (group - 1)) == 0 ? 128 / (int)group : 0;
    if (qbox && make_q_map(&qmap, p, qbox)) qbox = 0;
    cudaError_t e;
    if (TMA && (make_kv_map(&kmap, p.k, p, box) || make_kv_map(&vmap, p.v, p, box)))
        return launch<TYPE, DP, false>(p, 0, s);  // strides that no tensor map takes
    e = launch_pdl(k_attn_chunk<TYPE, DP, TMA>, dim3(grid), dim3(NTHREADS), F::SMEM, s, p, kmap, vmap, qmap, box, qbox);
    if (e == cudaSuccess) e = launch_pdl(k_attn_join_chunk<DP>, dim3(grid - 1, DP / JOIN_COLS), dim3(TR), 0, s, p);
    return (int)e;
}

// TMA where the pages allow it, else the copies: 16-byte copies are issued at 21 bytes per cycle and SM (about 1500 cycles
// a tile), close to the whole unit's time, and take four warps.
template <int TYPE, int DP>
int launch_pages(const AttnParams &p, cudaStream_t s) {
    const int box = kv_box(p.btd.d, 64);
    const bool strides = p.token_stride && p.block_stride && p.head_stride;
    return box && strides ? launch<TYPE, DP, true>(p, box, s) : launch<TYPE, DP, false>(p, 0, s);
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
        return p.head_dim <= 64 ? attn::launch_pages<T_BF16, 64>(p, s) : attn::launch_pages<T_BF16, 128>(p, s);
    return p.head_dim <= 64 ? attn::launch_pages<T_F16, 64>(p, s) : attn::launch_pages<T_F16, 128>(p, s);
}

}  // namespace ck
