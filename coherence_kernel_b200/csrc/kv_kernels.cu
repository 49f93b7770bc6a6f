// kv_kernels.cu -- the paged KV cache's bookkeeping: block tables and slot maps from request
// lengths, built on the device, and the write of new K/V rows through the slot map.
//
// A cache is n_blocks pages of block_tokens tokens.  Request r's token at position p lies in page
// table[r][p / block_tokens] at p % block_tokens; its slot is page * block_tokens + that.  Free pages
// are a stack: free[0 .. count).
#include "ck_launch.h"
#include "serve_common.cuh"

#include <cooperative_groups.h>

namespace ck {
namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int SAT = 1 << 30;  // sums saturate here: past every size that is accepted

// two operands of 0 .. SAT: their sum fits an unsigned int, not an int
CK_DEV int sat_add(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)SAT); }

// Inclusive scan of three saturating sums over the CTA; the running carry is returned in place.
struct Sum3 {
    int rows, need, back;
};
CK_DEV Sum3 add3(Sum3 a, Sum3 b) { return {sat_add(a.rows, b.rows), sat_add(a.need, b.need), sat_add(a.back, b.back)}; }
CK_DEV Sum3 shfl_up3(Sum3 v, int o) {
    return {__shfl_up_sync(0xffffffffu, v.rows, o), __shfl_up_sync(0xffffffffu, v.need, o),
            __shfl_up_sync(0xffffffffu, v.back, o)};
}
CK_DEV Sum3 warp_scan3(Sum3 v) {
    const int lane = threadIdx.x & 31;
    for (int o = 1; o < 32; o <<= 1) {
        const Sum3 u = shfl_up3(v, o);
        if (lane >= o) v = add3(v, u);
    }
    return v;
}

// the number of entries of a non-decreasing array that are <= key
CK_DEV int upper(const int *a, int n, int key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

struct ReqPlan {
    int len, rows, have, want;  // want: pages after the call if it is served
    bool fits;                  // its rows and its pages fit the caller's arrays
};

// The request lengths decide everything, so every CTA scans all of them -- a few loads per thread -- and no
// CTA waits for another's result.  The lengths and the sums over the requests (rows, pages needed, pages
// returned) stay in shared memory, and the rows, the new table entries and the returned pages are each a
// flat range that the grid's threads share out evenly, finding an element's request by binary search: one
// long prompt among a thousand decodes costs no more than its share.
//
// Taking a page never waits for a push either: the stack with the returned pages on top is read
// through the request that returned them, whose own table entries this call does not change.
//
// ALIAS: the lengths or the count are updated in place.  The CTAs are then one cluster, whose barrier
// comes between their reads and the writes.  Bound by latency (launch, the lengths, two scans, one lookup
// chain per row): 64 decodes 4.5 us, 1000 requests with 31,000 rows 8.3 us on 31 CTAs (15.4 us as one cluster of 8 that
// read the lengths from memory at each lookup).
template <bool ALIAS>
__global__ void __launch_bounds__(PLAN_THREADS) k_kv_plan(const KvPlanParams p) {
    extern __shared__ int sm[];
    const int n = (int)p.nreq;
    int *row_end = sm, *need_end = sm + n, *back_end = sm + 2 * n, *len_of = sm + 3 * n, *new_of = sm + 4 * n;
    __shared__ Sum3 warp_sum[PLAN_THREADS / 32];
    namespace cg = cooperative_groups;
    grid_dep_trigger_small();
    grid_dep_wait();
    const int count = min(max(p.count_in[0], 0), (int)p.n_blocks);
    const int cap = (int)(p.max_blocks * p.btd.d);  // below 2^30
    const auto req_plan = [&](int r) {
        ReqPlan q;
        q.len = len_of[r];
        const int nw = new_of[r];
        const int after = (int)min(max((int64_t)q.len + nw, (int64_t)0), (int64_t)SAT);
        q.rows = max(nw, 0);
        q.have = (int)p.btd.div((uint32_t)q.len + p.btd.d - 1);
        q.want = (int)p.btd.div((uint32_t)after + p.btd.d - 1);
        q.fits = q.rows > 0 && after <= cap && row_end[r] <= (int)p.ntok;
        return q;
    };
    Sum3 carry = {0, 0, 0};
    for (int base = 0; base < n; base += PLAN_THREADS) {
        const int r = base + (int)threadIdx.x;
        Sum3 v = {0, 0, 0};
        if (r < n) {
            len_of[r] = min(max(p.len_in[r], 0), cap);
            const int nw = p.new_tokens[r];
            new_of[r] = nw;
            v.rows = min(max(nw, 0), SAT);
            v.back = 0;
            if (nw < 0) {
                const int len = len_of[r], keep = max(len + max(nw, -SAT), 0);
                v.back = (int)(p.btd.div((uint32_t)len + p.btd.d - 1) - p.btd.div((uint32_t)keep + p.btd.d - 1));
            }
        }
        // rows and returned pages first: whether a request's rows fit decides whether the pages it needs count
        for (int pass = 0; pass < 2; ++pass) {
            if (pass == 1) {
                int need = 0;
                if (r < n) {
                    const ReqPlan q = req_plan(r);
                    if (q.fits) need = max(q.want - q.have, 0);
                }
                v = {0, need, 0};
            }
            Sum3 w = warp_scan3(v);
            if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = w;
            __syncthreads();
            Sum3 before = warp_scan3(warp_sum[threadIdx.x & 31]);
            const int wi = (int)(threadIdx.x >> 5);
            const Sum3 all = {__shfl_sync(0xffffffffu, before.rows, 31), __shfl_sync(0xffffffffu, before.need, 31),
                              __shfl_sync(0xffffffffu, before.back, 31)};
            const int src = max(wi - 1, 0);
            Sum3 prev = {__shfl_sync(0xffffffffu, before.rows, src), __shfl_sync(0xffffffffu, before.need, src),
                         __shfl_sync(0xffffffffu, before.back, src)};
            if (wi == 0) prev = {0, 0, 0};
            w = add3(add3(w, prev), carry);
            if (r < n) {
                if (pass == 0) row_end[r] = w.rows, back_end[r] = w.back;
                else need_end[r] = w.need;
            }
            carry = add3(carry, all);
            __syncthreads();
        }
    }
    const int back = n ? back_end[n - 1] : 0, need = n ? need_end[n - 1] : 0, rows = n ? row_end[n - 1] : 0;
    // at most n_blocks where the state is consistent; a count and lengths that are not may pass an int
    const int top = (int)min((unsigned)count + (unsigned)back, 0x7fffffffu);
    // requests are served in order while their pages last; the rest of the requests that need pages
    // get none.  taken: the largest of the running sums that fits
    int taken = need;
    if (need > top) {
        const int k = upper(need_end, n, top);
        taken = k ? need_end[k - 1] : 0;
    }
    const auto served = [&](const ReqPlan &q, int r) {
        return q.fits && (q.want <= q.have || need_end[r] <= top);
    };
    // page number k of this call, counting down from the stack's top
    const auto page = [&](int k) {
        const int at = top - 1 - k;
        if (at < count) return at >= 0 ? p.free_blocks[at] : -1;
        const int i = at - count, r = upper(back_end, n, i);
        if (r >= n) return -1;
        const ReqPlan q = req_plan(r);
        return p.table[(uint64_t)r * p.table_stride + q.want + (i - (back_end[r] - (q.have - q.want)))];
    };
    const int gt = (int)(blockIdx.x * PLAN_THREADS + threadIdx.x), gn = (int)(gridDim.x * PLAN_THREADS);

    // slots and positions of the rows
    const int live = min(rows, (int)p.ntok);
    for (int t = gt; t < (int)p.ntok; t += gn) {
        int64_t slot = -1;
        int pos = -1;
        if (t < live) {
            const int r = upper(row_end, n, t);
            const ReqPlan q = req_plan(r);
            if (served(q, r)) {
                pos = q.len + t - (row_end[r] - q.rows);
                const int b = (int)p.btd.div((uint32_t)pos);
                const int pg = b < q.have ? p.table[(uint64_t)r * p.table_stride + b]
                                          : page(need_end[r] - (q.want - q.have) + b - q.have);
                if (pg >= 0 && pg < (int)p.n_blocks) slot = (int64_t)pg * p.btd.d + (pos - b * (int)p.btd.d);
            }
        }
        p.slots[t] = slot;
        p.positions[t] = pos;
    }
    // new table entries
    for (int k = gt; k < taken; k += gn) {
        const int r = upper(need_end, n, k);
        const ReqPlan q = req_plan(r);
        p.table[(uint64_t)r * p.table_stride + q.have + (k - (need_end[r] - (q.want - q.have)))] = page(k);
    }
    // returned pages that nobody took: pushed above the old top
    for (int i = gt; i < top - taken - count; i += gn) {
        const int r = upper(back_end, n, i);
        const ReqPlan q = req_plan(r);
        if (count + i < (int)p.n_blocks)
            p.free_blocks[count + i] =
                p.table[(uint64_t)r * p.table_stride + q.want + (i - (back_end[r] - (q.have - q.want)))];
    }
    for (int r = gt; r <= n; r += gn) p.q_start[r] = r ? min(row_end[r - 1], (int)p.ntok) : 0;
    if (ALIAS) cg::this_cluster().sync();  // every CTA has read the lengths and the count
    for (int r = gt; r < n; r += gn) {
        const ReqPlan q = req_plan(r);
        const int nw = new_of[r];
        const bool ok = served(q, r);
        const int after = (int)max((int64_t)q.len + nw, (int64_t)0);
        const int len = nw > 0 && !ok ? q.len : after;
        p.kv_len[r] = nw > 0 && !ok ? 0 : len;
        p.len_out[r] = len;
    }
    if (gt == 0) p.count_out[0] = min(top - taken, (int)p.n_blocks);
}

// K/V rows into the cache: one thread moves eight elements of one row of K or V per step, so a
// warp's reads and writes are whole rows of 16-byte pieces.  Nothing is kept between elements: HBM
// (many rows) or one read-write round trip (few) is the bound: 8192 tokens of 8 x 128, bf16, 8.3 us (57.6 MB); 64 from f32 1.6 us.
template <int IN>
__global__ void __launch_bounds__(256) k_kv_append(const KvAppendParams p) {
    grid_dep_trigger_small();
    grid_dep_wait();
    const uint32_t vec_row = p.row_div.d;  // eight-element pieces of a token's K (or V)
    const uint32_t total = 2 * p.ntok * vec_row;
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) {
        const uint32_t row = p.row_div.div(i), c = i - row * vec_row;
        const uint32_t t = row >> 1;
        const bool is_v = row & 1;
        const int64_t slot = p.slots[t];
        if (slot < 0 || slot >= p.n_slots) continue;
        const uint32_t h = p.head_div.div(c), d = (c - h * p.head_div.d) * 8;
        const Raw8 raw = load_raw8(is_v ? p.v : p.k, (uint64_t)t * (is_v ? p.v_stride : p.k_stride) + c * 8, IN);
        const uint32_t b = p.btd.div((uint32_t)slot);
        const uint64_t at = b * p.block_stride + ((uint32_t)slot - b * p.btd.d) * p.token_stride + h * p.head_stride + d;
        void *cache = is_v ? p.v_cache : p.k_cache;
        float v[8];
        raw8_to_float(raw, IN, v);
        store8(cache, at, p.cache_type, v);
    }
}

}  // namespace

int launch_kv_plan(const KvPlanParams &p, cudaStream_t s) {
    const size_t smem = (size_t)p.nreq * 20;
    static unsigned long long done = 0;
    if (attr_pending(done)) {
        cudaError_t e = cudaFuncSetAttribute(k_kv_plan<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             KV_PLAN_MAX_REQUESTS * 20);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(k_kv_plan<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     KV_PLAN_MAX_REQUESTS * 20);
        if (e != cudaSuccess) return (int)e;
        attr_mark(done);
    }
    // a CTA per 1024 rows or requests; one cluster (of 1, 2, 4 or 8) where the state is updated in place
    const bool alias = p.len_out == p.len_in || p.count_out == p.count_in;
    const uint32_t most = p.ntok > p.nreq ? p.ntok : p.nreq, want = (most + PLAN_THREADS - 1) / PLAN_THREADS;
    uint32_t ctas = want < 1 ? 1 : want < SMS ? want : SMS;
    if (alias) ctas = want <= 1 ? 1 : want <= 2 ? 2 : want <= 4 ? 4 : 8;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = alias ? ctas : 1;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(PLAN_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)(alias ? cudaLaunchKernelEx(&cfg, k_kv_plan<true>, p) : cudaLaunchKernelEx(&cfg, k_kv_plan<false>, p));
}

int launch_kv_append(const KvAppendParams &p, int in_type, cudaStream_t s) {
    const uint32_t want = (2 * p.ntok * p.row_div.d + 255) / 256;
    const dim3 grid(want < 8 * SMS ? want : 8 * SMS);
    switch (in_type) {
        case T_F32: return (int)launch_pdl(k_kv_append<T_F32>, grid, dim3(256), 0, s, p);
        case T_F16: return (int)launch_pdl(k_kv_append<T_F16>, grid, dim3(256), 0, s, p);
        default: return (int)launch_pdl(k_kv_append<T_BF16>, grid, dim3(256), 0, s, p);
    }
}

}  // namespace ck
