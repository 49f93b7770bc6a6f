// attn_sched.cuh -- how the attention kernels share their work out over a fixed number of CTAs.
//
// An item is one tile of TR rows (rows = tokens x the query heads of one K/V head, token-major) of
// one request and K/V head; a unit is KC consecutive keys of an item.  An item also counts for EXTRA
// units without keys at its end: what its queries' load and its epilogue cost, so that a CTA of many
// short items gets no more work than one of a long one (64 ragged decodes, 1 to 8192 tokens: the
// slowest CTA took twice the median's time).  Units are numbered request by request, tile by tile,
// head by head, key chunk by key chunk, and CTA c of C takes units [c U / C, (c + 1) U / C): the split
// depends on the lengths alone, so ragged batches, one long request and many short ones all fill the
// GPU evenly and results do not depend on timing.  An item that spans CTAs leaves one partial result
// per CTA (running maximum, sum, unnormalised output), joined in CTA order: in the few-row form by the
// CTA that brings the last part, whoever it is (one launch less: 2 us of a small call's host time), in
// the chunk form, whose parts are 256 rows, by a second kernel that spreads them over the GPU (17
// ragged requests 55 us; in the last CTA 69).
//
// The lengths are device data: every CTA sums the units of all requests itself (a few loads per
// thread) instead of waiting for a planning kernel.
#pragma once
#include "ck_launch.h"
#include "serve_common.cuh"

namespace ck {
namespace attn {

struct Req {
    int q0, nq, kl;  // first row of q, new tokens, visible cache length
};
CK_DEV Req load_req(const AttnParams &p, int r) {
    Req q;
    const int a = min(max(p.q_start[r], 0), (int)p.ntok), b = min(max(p.q_start[r + 1], a), (int)p.ntok);
    q.q0 = a;
    q.nq = b - a;
    q.kl = (int)min((int64_t)max(p.kv_len[r], 0), (int64_t)p.max_blocks * p.btd.d);
    return q;
}

struct Geo {
    int lo, hi, nch;  // keys [lo, hi) of the tile and its chunks (at least one, so that empty rows are written)
};
// Keys a tile of rows [row, row + TR) sees: the last row's upper bound, the first row's lower one (down to a multiple
// of ALIGN).
template <int TR, int KC, int ALIGN>
CK_DEV Geo tile_geo(const AttnParams &p, const Req &q, int t) {
    const int rows = q.nq * (int)p.gd.d;
    const int first = t * TR, last = min(first + TR, rows) - 1;
    const int base = q.kl - q.nq;  // position of the request's first new token
    Geo g;
    g.hi = p.causal ? min(q.kl, base + (int)p.gd.div(last) + 1) : q.kl;
    g.lo = p.window ? max(0, base + (int)p.gd.div(first) - p.window + 1) & ~(ALIGN - 1) : 0;
    if (g.hi <= g.lo) {
        g.lo = g.hi = 0;
        g.nch = 1;
    } else {
        g.nch = (g.hi - g.lo + KC - 1) / KC;
    }
    return g;
}

struct Pos {
    int r, t, h, c;
};

// The kind of request a kernel takes: few rows, or many (CHUNK).
template <int TR, int KC, bool CHUNK>
struct Sched {
    static constexpr int ALIGN = CHUNK ? 64 : 16;
    static constexpr int EXTRA = CHUNK ? 3 : 2;
    static constexpr int PARTS = 128;
    static CK_DEV int tiles(const AttnParams &p, const Req &q) {
        const int rows = q.nq * (int)p.gd.d;
        if (CHUNK ? rows < (int)p.row_split : rows >= (int)p.row_split) return 0;
        return (rows + TR - 1) / TR;
    }
    // units of request r, which is returned in q (all 32 lanes of a warp call this together, each with its own request)
    static CK_DEV long long units(const AttnParams &p, int r, Req &q) {
        q = {0, 0, 0};
        if (r < (int)p.nreq) q = load_req(p, r);
        const int nt = r < (int)p.nreq ? tiles(p, q) : 0;
        long long n = 0;
        if (nt <= 8)
            for (int t = 0; t < nt; ++t) n += tile_geo<TR, KC, ALIGN>(p, q, t).nch + EXTRA;
        // requests of many tiles: the warp's lanes share them out
        for (uint32_t todo = __ballot_sync(0xffffffffu, nt > 8); todo; todo &= todo - 1) {
            const int src = __ffs(todo) - 1;
            const Req w = {0, __shfl_sync(0xffffffffu, q.nq, src), __shfl_sync(0xffffffffu, q.kl, src)};
            const int wt = __shfl_sync(0xffffffffu, nt, src);
            long long part = 0;
            for (int t = threadIdx.x & 31; t < wt; t += 32) part += tile_geo<TR, KC, ALIGN>(p, w, t).nch + EXTRA;
            for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
            if ((int)(threadIdx.x & 31) == src) n = part;
        }
        return n * (int)p.n_kv;
    }

    struct Shared {
        long long warp_sum[32];
        int warp_items[32];
        long long before;
        Pos pos;
        Geo geo;
        Req req;
    };
    // exclusive prefix of v over the CTA; `all` receives the sum, `items` that of the threads' items
    static CK_DEV long long scan(long long v, Shared &sh, long long &all, int &items) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
        long long s = v;
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        items = (int)__reduce_add_sync(0xffffffffu, (unsigned)items);
        if (lane == 31) {
            sh.warp_sum[w] = s;
            sh.warp_items[w] = items;
        }
        __syncthreads();
        long long before = 0;
        all = 0;
        items = 0;
        for (int i = 0; i < nw; ++i) {
            if (i < w) before += sh.warp_sum[i];
            all += sh.warp_sum[i];
            items = min(items + sh.warp_items[i], 1 << 20);
        }
        __syncthreads();
        return before + s - v;
    }
    // U c / C; a 64-bit division is a hundred instructions, and few batches need it (C < 512)
    static CK_DEV long long start(long long U, int C, int c) {
        return U < 1 << 22 ? (long long)((uint32_t)U * (uint32_t)c / (uint32_t)C) : U * c / C;
    }

    // Called by the whole CTA.  Finds the total U, the CTAs that take part C -- at most one a unit, and PARTS an item
    // on average: joining a part costs about a tenth of a unit -- and the position of unit start(cta); returns false
    // when cta takes no part.
    static CK_DEV bool find(const AttnParams &p, Shared &sh, int grid, int cta, long long &U, int &C, Pos &pos, Geo &geo) {
        const int n = (int)p.nreq, bd = (int)blockDim.x;
        Req q;
        long long mine = units(p, threadIdx.x, q), sum = mine;
        int items = (int)min((long long)tiles(p, q) * p.n_kv, 1ll << 16);
        for (int b = bd; b < n; b += bd) {
            Req o;
            sum += units(p, b + (int)threadIdx.x, o);
            items = min(items + (int)min((long long)tiles(p, o) * p.n_kv, 1ll << 16), 1 << 16);
        }
        long long ex = scan(sum, sh, U, items);
        C = (int)(U < grid ? U : grid);
        C = min(C, PARTS * items);
        if (cta >= C) return false;
        const long long u = start(U, C, cta);
        if (n > bd) {  // more requests than threads: once more, block by block
            long long base = 0, all = 0;
            for (int b = 0;; b += bd) {
                mine = units(p, b + (int)threadIdx.x, q);
                ex = base + scan(mine, sh, all, items);
                if (u >= ex && u < ex + mine) sh.pos.r = b + (int)threadIdx.x;
                if (u < base + all) break;
                base += all;
            }
        } else if (u >= ex && u < ex + mine) {
            sh.pos.r = (int)threadIdx.x;
        }
        if (u >= ex && u < ex + mine) {  // one thread: its request holds the unit
            sh.before = u - ex;
            sh.req = q;
            if (tiles(p, q) == 1) place(p, sh, q, 0, tile_geo<TR, KC, ALIGN>(p, q, 0), u - ex);
        }
        __syncthreads();
        const int nt = tiles(p, sh.req);
        if (nt > 1) {
            if (threadIdx.x < 32) {  // the tile of the request: 32 at a time
                const int lane = threadIdx.x;
                long long v = sh.before;
                q = sh.req;
                for (int tb = 0; tb < nt; tb += 32) {
                    const int t = tb + lane;
                    Geo g = {0, 0, 0};
                    if (t < nt) g = tile_geo<TR, KC, ALIGN>(p, q, t);
                    const long long m = t < nt ? (long long)(g.nch + EXTRA) * p.n_kv : 0;
                    long long s = m;
                    for (int o = 1; o < 32; o <<= 1) {
                        const long long x = __shfl_up_sync(0xffffffffu, s, o);
                        if (lane >= o) s += x;
                    }
                    const long long tot = __shfl_sync(0xffffffffu, s, 31);
                    if (v < tot) {
                        if (v >= s - m && v < s) place(p, sh, q, t, g, v - (s - m));
                        break;
                    }
                    v -= tot;
                }
            }
            __syncthreads();
        }
        pos = sh.pos;
        geo = sh.geo;
        return true;
    }
    static CK_DEV void place(const AttnParams &p, Shared &sh, const Req &q, int t, const Geo &g, long long in) {
        const uint32_t per = (uint32_t)(g.nch + EXTRA);
        sh.pos.t = t;
        sh.pos.h = in < 1ll << 32 ? (int)((uint32_t)in / per) : (int)(in / per);
        sh.pos.c = (int)(in - (long long)sh.pos.h * per);
        sh.geo = g;
    }

    // A walk over a CTA's consecutive units, item by item: units c0 .. c1 - 1 (with keys) of the item are the CTA's.
    struct Items {
        Pos at;
        Req q;
        Geo g;
        int nt, left, c0, c1;
        long long first;  // the item's first unit
        // false if the CTA has no unit with keys
        CK_DEV bool set(const AttnParams &p, const Shared &sh, int n, long long u0 = 0) {
            first = u0 - sh.pos.c;
            at = sh.pos;
            g = sh.geo;
            q = sh.req;
            nt = tiles(p, q);
            left = n;
            c0 = at.c;
            c1 = min(g.nch, c0 + left);
            return c0 < g.nch || next(p);
        }
        CK_DEV bool whole() const { return c0 == 0 && c1 == g.nch; }
        // the next item; false at the end of the CTA's range
        CK_DEV bool next(const AttnParams &p) {
            left -= g.nch + EXTRA - c0;
            first += g.nch + EXTRA;
            if (left <= 0) return false;
            if (++at.h >= (int)p.n_kv) {
                at.h = 0;
                if (++at.t >= nt) {
                    at.t = 0;
                    do {
                        if (++at.r >= (int)p.nreq) return false;
                        q = load_req(p, at.r);
                        nt = tiles(p, q);
                    } while (nt == 0);
                }
                g = tile_geo<TR, KC, ALIGN>(p, q, at.t);
            }
            c0 = 0;
            c1 = min(g.nch, left);
            return true;
        }
    };

    // The parts of an item that spans CTAs: those of CTAs cta .. cta + n - 1, in each CTA's slot 0 except, where the
    // item is not the first with keys in the first CTA's range, slot 1 there.
    struct Joint {
        int cta, n, slot0;
        CK_DEV size_t slot(int i) const { return (size_t)(cta + i) * 2 + (i == 0 ? slot0 : 0); }
    };
    static CK_DEV Joint joint(const Items &it, long long U, int C) {
        // the CTA of unit u is the largest c with U c / C <= u, that is c <= (C (u + 1) - 1) / U
        const long long a = it.first, b = a + it.g.nch;
        Joint j;
        j.cta = (int)((C * (a + 1) - 1) / U);
        j.n = (int)((C * b - 1) / U) - j.cta + 1;
        j.slot0 = start(U, C, j.cta) >= a - EXTRA ? 0 : 1;  // a start behind the last item's keys is as good as a
        return j;
    }

    // What the joining kernel needs of each CTA's start, left in the workspace by the CTA.
    static CK_DEV void leave_cut(const AttnParams &p, long long U, int C, const Pos &at, const Geo &g) {
        if (threadIdx.x == 0) {
            if (blockIdx.x == 0) {
                p.cuts->units = U;
                p.cuts->ctas = C;
            }
            if ((int)blockIdx.x < C) p.cuts->at[blockIdx.x] = make_int4(at.r, at.t, at.h, at.c);
            if ((int)blockIdx.x < C) p.cuts->chunks[blockIdx.x] = g.nch;
        }
    }
};

// An item that spans CTAs, seen from boundary j (the start of CTA j's units): found at its first cut only.
// Its parts are those of CTAs first .. first + n - 1, in each CTA's slot 0 except, where the item is not the first
// with keys in the first CTA's range, slot 1 there.
struct Cut {
    Pos at;
    int first, n, slot0;
    CK_DEV size_t slot(int i) const { return (size_t)(first + i) * 2 + (i == 0 ? slot0 : 0); }
};
template <class S>
CK_DEV bool find_joint(const AttnParams &p, int j, Cut &o) {
    const long long U = p.cuts->units;
    const int C = p.cuts->ctas;
    if (j >= C) return false;
    const int4 v = p.cuts->at[j];
    const long long u = U * j / C, a = u - v.w, b = a + p.cuts->chunks[j];
    const long long before = U * (j - 1) / C;
    // the cut is an item's start, or behind its last keys, or not its first
    if (v.w == 0 || v.w >= p.cuts->chunks[j] || before > a) return false;
    o.at = {v.x, v.y, v.z, v.w};
    o.first = j - 1;
    o.slot0 = before >= a - S::EXTRA ? 0 : 1;  // a start behind the last item's keys is as good as a
    // the CTA of unit b - 1: the largest c with U c / C <= b - 1, that is c <= (C b - 1) / U
    o.n = (int)(((long long)C * b - 1) / U) - o.first + 1;
    return true;
}

// TMA loads of a cache: a 4D map (dim, head, token of a page, page), a box of 64 dims (128 bytes, swizzled) of one
// head for `box` consecutive tokens of one page.  Pages whose token count is a multiple of 8 qualify; a page past
// the last reads as zeros.
CK_DEV void tma_load_kv(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int d, int head, int tok, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(d), "r"(head), "r"(tok), "r"(page)
        : "memory");
}
inline int kv_box(uint32_t block_tokens, int most) {
    int b = most;
    while (b >= 8 && block_tokens % b) b >>= 1;
    return b >= 8 ? b : 0;
}
inline int encode_map(CUtensorMap *m, const void *base, int type, cuuint32_t rank, const cuuint64_t *dims,
                      const cuuint64_t *strides, const cuuint32_t *box) {
    using Fn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                            const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Fn enc = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<Fn>(f)
                   : nullptr;
    }();
    if (!enc) return CK_ERR_NODEV;
    const cuuint32_t one[4] = {1, 1, 1, 1};
    const CUresult r = enc(m, type == T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                           const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : CK_ERR_ARG;
}
inline int make_kv_map(CUtensorMap *m, const void *base, const AttnParams &p, int box) {
    const cuuint64_t dims[4] = {p.head_dim, p.n_kv, p.btd.d, p.n_blocks};
    const cuuint64_t strides[3] = {p.head_stride * 2, p.token_stride * 2, p.block_stride * 2};
    const cuuint32_t box4[4] = {64, 1, (cuuint32_t)box, 1};
    return encode_map(m, base, p.cache_type, 4, dims, strides, box4);
}

// The keys that row's token may see: [lo, hi).
CK_DEV void row_limits(const AttnParams &p, const Req &q, int row, int &lo, int &hi) {
    const int pos = q.kl - q.nq + (int)p.gd.div((uint32_t)row);
    hi = p.causal ? min(q.kl, pos + 1) : q.kl;
    lo = p.window ? max(0, pos - p.window + 1) : 0;
}

// Element offset of key j of request r in the cache (head 0), or -1 for a page outside the cache.
CK_DEV int64_t key_offset(const AttnParams &p, int r, int j) {
    const uint32_t b = p.btd.div((uint32_t)j);
    const int pg = p.table[(uint64_t)r * p.table_stride + b];
    if (pg < 0 || pg >= (int)p.n_blocks) return -1;
    return (int64_t)((uint64_t)pg * p.block_stride + ((uint32_t)j - b * p.btd.d) * p.token_stride);
}

CK_DEV bool finite16(uint16_t b, int type) {
    const uint16_t m = type == T_BF16 ? 0x7F80 : 0x7C00;
    return (b & m) != m;
}
CK_DEV float value16(uint16_t b, int type) {
    return type == T_BF16 ? bf16_bits_to_float(b) : __half2float(__ushort_as_half(b));
}
// Where some rows of a tile see a key and others do not, the matrix product takes V's infinities and
// NaNs as zeros (0 x inf would reach the rows that do not see them); this is what they add to the
// rows that do: the sum of the non-finite V[j][d] over the visible j of [j0, j1), in the steps of `step` keys that reach
// outside [all_lo, all_hi), the keys that every row sees.  Rare, so a call; scalars only, so that it keeps nothing
// of the caller's in memory.
static __device__ __noinline__ float nonfinite_v(const AttnParams &p, int r, int h, int d, int j0, int j1, int step,
                                                 int all_lo, int all_hi, int lo, int hi) {
    float s = 0.0f;
    if (d >= (int)p.head_dim) return s;
    for (int b = j0; b < j1; b += step) {
        if (b >= all_lo && b + step <= all_hi) continue;
        for (int j = max(b, lo); j < min(min(b + step, j1), hi); ++j) {
            const int64_t at = key_offset(p, r, j);
            if (at < 0) continue;
            const uint16_t w = static_cast<const uint16_t *>(p.v)[at + (int64_t)(h * p.head_stride) + d];
            if (!finite16(w, p.cache_type)) s += value16(w, p.cache_type);
        }
    }
    return s;
}

CK_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LN2 = 0.69314718055994531f;

}  // namespace attn
}  // namespace ck
