// page_plan.cu - one step's page plan of a paged key / value cache: pages of finished rows back onto the stack of free pages, pages
// for the rows that grow, and every new token's cache slot, position and row.
//
// All of it follows from three running sums over the rows: the new tokens, the pages that rows need and the pages that finished
// rows give back.  Every block makes the three sums of all rows itself (at most 2048 rows, two a thread), keeps them in shared memory
// and then takes its share of the tokens and pages, each of which finds its row by bisection: no block waits for another one's
// result.  What a call may write over its own inputs (lengths, free count) is written after a cluster barrier, when every block has
// read them; that is why the blocks of a call are one cluster.  Pages are popped where they lie: page k of the step is entry
// have - 1 - k of the stack with the given-back pages on top, so nothing is pushed that this step pops again.
//
// Bound by latency: a chain of loads of the rows, the scan, one or two dependent loads for a token's page.  On a B200: 32 rows, a token each,
// 3.8 us; 512 rows with 16512 places 7.5 us in a cluster of eight blocks, 18.9 in one block.
#include "common.cuh"
#include "pdl.cuh"

#include <cooperative_groups.h>

namespace bsx {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kRowsPerThread = BSX_PAGED_MAX_ROWS / kPlanThreads;

struct PagePlanParams {
    const int32_t* seq_len;
    const int32_t* n_new;
    int32_t* table;
    int64_t table_stride;
    int32_t* free_list;
    const int32_t* free_count;
    int32_t* seq_len_out;
    int32_t* free_count_out;
    int32_t* cu_new;
    int64_t* slot;
    int32_t* pos;
    int32_t* row;
    int32_t* status;
    int32_t n_rows, page_shift, max_pages, free_cap, cap_tokens;
};

// first index whose running sum is above v (n when none is)
__device__ __forceinline__ int row_of(const uint32_t* ends, int n, uint32_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > v) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Sums stop at 2^31 - 1, past every capacity they are compared with; such a sum of non-negative terms is associative, as the scan needs.
__device__ __forceinline__ uint32_t add_capped(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PagePlanParams p) {
    namespace cg = cooperative_groups;
    __shared__ uint32_t tok_end[BSX_PAGED_MAX_ROWS], need_end[BSX_PAGED_MAX_ROWS], back_end[BSX_PAGED_MAX_ROWS];
    __shared__ int32_t length[BSX_PAGED_MAX_ROWS];
    __shared__ uint8_t served[BSX_PAGED_MAX_ROWS];
    __shared__ uint32_t sums[3][32];
    __shared__ uint32_t popped_s;
    __shared__ int32_t trouble;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.n_rows, shift = p.page_shift;
    const int page = 1 << shift;
    const int64_t longest = (int64_t) p.max_pages << shift;
    pdl_wait();
    if (tid == 0) {
        popped_s = 0;
        trouble = 0;
    }

    // a thread's rows, and their three sums
    uint32_t tok[kRowsPerThread], need[kRowsPerThread], back[kRowsPerThread];
    int32_t len[kRowsPerThread], grow[kRowsPerThread];
    uint8_t ok[kRowsPerThread];
    int32_t why = 0;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const int r = tid * kRowsPerThread + i;
        tok[i] = need[i] = back[i] = 0;
        len[i] = grow[i] = 0;
        ok[i] = 0;
        if (r >= n) continue;
        len[i] = p.seq_len[r];
        grow[i] = p.n_new[r];
        const bool sound = len[i] >= 0 && len[i] <= longest;
        const int32_t held = sound ? (int32_t) (((int64_t) len[i] + page - 1) >> shift) : 0;
        if (!sound) why |= BSX_PAGED_BAD_STATE;
        if (grow[i] < 0) {
            back[i] = (uint32_t) held;
        } else {
            tok[i] = (uint32_t) grow[i];
            const int64_t after = (int64_t) len[i] + grow[i];
            if (sound && after > longest) why |= BSX_PAGED_TOO_LONG;
            if (sound && after <= longest) {
                ok[i] = 1;
                need[i] = (uint32_t) (((after + page - 1) >> shift) - held);
            }
        }
    }
    uint32_t mine[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        mine[0] = add_capped(mine[0], tok[i]);
        mine[1] = add_capped(mine[1], need[i]);
        mine[2] = add_capped(mine[2], back[i]);
    }
    uint32_t incl[3] = {mine[0], mine[1], mine[2]};
#pragma unroll
    for (int q = 0; q < 3; ++q) {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t o = __shfl_up_sync(kFull, incl[q], d);
            if (lane >= d) incl[q] = add_capped(incl[q], o);
        }
        if (lane == 31) sums[q][warp] = incl[q];
    }
    __syncthreads();
    if (warp < 3) {
        uint32_t v = sums[warp][lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t o = __shfl_up_sync(kFull, v, d);
            if (lane >= d) v = add_capped(v, o);
        }
        sums[warp][lane] = v;
    }
    __syncthreads();
    uint32_t run[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        const uint32_t before = __shfl_up_sync(kFull, incl[q], 1);
        run[q] = add_capped(warp ? sums[q][warp - 1] : 0u, lane ? before : 0u);
    }
    const uint32_t n_tok = sums[0][31], n_back = sums[2][31];

    const int32_t count_in = *p.free_count;
    const int32_t count = min(max(count_in, 0), p.free_cap);
    const uint32_t room = (uint32_t) (p.free_cap - count);
    if (count != count_in || n_back > room) why |= BSX_PAGED_BAD_STATE;
    const uint32_t have = (uint32_t) count + min(n_back, room);
    uint32_t last = 0;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const int r = tid * kRowsPerThread + i;
        run[0] = add_capped(run[0], tok[i]);
        run[1] = add_capped(run[1], need[i]);
        run[2] = add_capped(run[2], back[i]);
        if (r >= n) continue;
        const bool places = run[0] <= (uint32_t) p.cap_tokens || tok[i] == 0;
        const bool pages = run[1] <= have || need[i] == 0;
        if (ok[i] && !places) why |= BSX_PAGED_NO_PLACES;
        if (ok[i] && !pages) why |= BSX_PAGED_NO_PAGES;
        ok[i] = ok[i] && places && pages;
        if (ok[i] && need[i]) last = max(last, run[1]);
        tok_end[r] = run[0];
        need_end[r] = run[1];
        back_end[r] = run[2];
        length[r] = len[i];
        served[r] = ok[i];
    }
    last = __reduce_max_sync(kFull, last);
    why = __reduce_or_sync(kFull, why);
    if (lane == 0) {
        if (last) atomicMax(&popped_s, last);
        if (why) atomicOr(&trouble, why);
    }
    __syncthreads();
    const uint32_t popped = popped_s, left = have - popped;

    auto given_back = [&](uint32_t j) {
        const int r = row_of(back_end, n, j);
        return p.table[r * p.table_stride + (j - (r ? back_end[r - 1] : 0u))];
    };
    auto popped_page = [&](uint32_t k) {
        const uint32_t at = have - 1 - k;
        return at < (uint32_t) count ? p.free_list[at] : given_back(at - count);
    };
    const uint32_t first = blockIdx.x * kPlanThreads + tid, step = gridDim.x * kPlanThreads;
    for (uint32_t t = first; t < (uint32_t) p.cap_tokens; t += step) {
        int64_t slot = -1;
        int32_t at = 0, of = -1;
        const int r = t < n_tok ? row_of(tok_end, n, t) : n;
        if (r < n && served[r]) {
            of = r;
            at = length[r] + (int32_t) (t - (r ? tok_end[r - 1] : 0u));
            const int32_t held = (length[r] + page - 1) >> shift, i = at >> shift;
            const int32_t id = i < held ? p.table[r * p.table_stride + i] : popped_page((r ? need_end[r - 1] : 0u) + (uint32_t) (i - held));
            slot = ((int64_t) id << shift) + (at & (page - 1));
        }
        p.slot[t] = slot;
        p.pos[t] = at;
        p.row[t] = of;
    }
    for (uint32_t k = first; k < popped; k += step) {
        const int r = row_of(need_end, n, k);
        const int32_t held = (length[r] + page - 1) >> shift;
        p.table[r * p.table_stride + held + (k - (r ? need_end[r - 1] : 0u))] = popped_page(k);
    }
    for (uint32_t j = first; (uint32_t) count + j < left; j += step) p.free_list[count + j] = given_back(j);

    if (gridDim.x > 1) cg::this_cluster().sync();   // every block has read the lengths and the free count
    if (blockIdx.x) return;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const int r = tid * kRowsPerThread + i;
        if (r >= n) continue;
        p.cu_new[r + 1] = (int32_t) min(tok_end[r], (uint32_t) p.cap_tokens);
        const bool sound = len[i] >= 0 && len[i] <= longest;
        p.seq_len_out[r] = !sound ? len[i] : grow[i] < 0 ? 0 : ok[i] ? len[i] + grow[i] : len[i];
    }
    if (tid == 0) {
        p.cu_new[0] = 0;
        *p.free_count_out = (int32_t) left;
        if (p.status && trouble) atomicOr(p.status, trouble);
    }
}

}  // namespace
}  // namespace bsx

using namespace bsx;

extern "C" int32_t bsx_page_plan(const int32_t* seq_len, const int32_t* n_new, int32_t n_rows, int32_t page_size, int32_t* block_table,
                                 int64_t table_stride, int32_t max_pages, int32_t* free_list, int32_t free_cap, const int32_t* free_count,
                                 int32_t cap_tokens, int32_t* seq_len_out, int32_t* free_count_out, int32_t* cu_new, int64_t* slot, int32_t* pos,
                                 int32_t* row, int32_t* status, void* stream) {
    if (!stream) return BSX_E_STREAM;
    if (n_rows <= 0 || max_pages <= 0 || table_stride < max_pages || free_cap < 0 || cap_tokens < 0 || page_size < 8 || page_size > 256 ||
        (page_size & (page_size - 1)))
        return BSX_E_GEOMETRY;
    if (n_rows > BSX_PAGED_MAX_ROWS || cap_tokens > BSX_PAGED_MAX_TOKENS || (int64_t) max_pages * page_size > BSX_PAGED_MAX_KEYS || free_cap > 1 << 30)
        return BSX_E_LIMIT;
    if (!seq_len || !n_new || !block_table || !free_count || !seq_len_out || !free_count_out || !cu_new || (free_cap && !free_list) ||
        (cap_tokens && (!slot || !pos || !row)))
        return BSX_E_POINTER;
    int shift = 3;
    while ((1 << shift) != page_size) ++shift;
    const PagePlanParams p{seq_len,  n_new, block_table, table_stride, free_list, free_count, seq_len_out, free_count_out, cu_new,
                           slot,     pos,   row,         status,       n_rows,    shift,      max_pages,   free_cap,       cap_tokens};
    // the largest portable cluster, or fewer blocks where each would have less than one token a thread
    int blocks = (cap_tokens + kPlanThreads - 1) / kPlanThreads;
    blocks = blocks > 8 ? 8 : blocks < 1 ? 1 : blocks;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned) blocks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // as launch_early
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) blocks);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.stream = (cudaStream_t) stream;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    (void) cudaLaunchKernelEx(&cfg, page_plan_kernel, p);
    return launch_status();
}
