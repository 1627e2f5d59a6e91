// One step's pages from a free list in device memory (tllm_paged_plan).
//
// Per request: have = ceil(len / P) pages before, need = ceil((len + new) / P) behind; three running sums over the requests (tokens, pages
// taken, pages returned) say where a request's rows, its new pages in the ring and its returned pages go.  Everything else is
// independent: row t finds its request by bisection of the sums, and a page that is new is table entry j of its request, taken
// from ring[head + taken before + j - have] - the row knows that without reading what another workgroup writes.  So ONE launch does it
// all: every workgroup forms the sums itself (4096 requests: 32 KB from L2 and one block scan), keeps them in LDS and fills its share of
// rows.  The row whose token opens a page writes the table entry (a new page always starts with a token of this step).
// Bound by latency, not by bytes: lengths -> scan -> ring / table -> store (16 requests 4.1 us; 512 requests with 54000 rows, 0.5 MB, 6.0 us: half
// of that is the launch).
#include "dev_utils.h"
#include "launch_util.h"
#include "serving_kernels.h"
#include <algorithm>

namespace tllm
{
namespace kernels
{
using namespace dev;

namespace
{
constexpr int kThreads = 1024, kWaves = kThreads / 64, kPer = kPlanMaxSeqs / kThreads, kRowsPerGroup = 1024;

enum Part : int
{
    PART_ALL = 0,   // one workgroup, or a state that is written elsewhere than it is read
    PART_ROWS = 1,  // several workgroups and a state that is updated in place: everything but the state ..
    PART_STATE = 2, // .. and the state, by one workgroup behind them
};

struct Three
{
    uint32_t a, b, c;
};

__device__ __forceinline__ Three wave_scan(Three v) // inclusive, over the wave
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
    {
        const uint32_t a = __shfl_up(v.a, d, 64), b = __shfl_up(v.b, d, 64), c = __shfl_up(v.c, d, 64);
        if (lane >= d)
        {
            v.a += a;
            v.b += b;
            v.c += c;
        }
    }
    return v;
}

__global__ __launch_bounds__(kThreads) void plan_kernel(const tllm_paged_plan_params_t p, const int shift, const int part)
{
    extern __shared__ uint32_t lds[]; // [n_seqs + 1] rows before, [n_seqs] pages taken before, pages returned before, lens, new_lens
    __shared__ Three wave_sum_[kWaves];
    __shared__ int bad_;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.n_seqs;
    uint32_t* const rows_before = lds;
    uint32_t* const taken_before = lds + n + 1;
    uint32_t* const given_before = taken_before + n;
    int32_t* const len_of = reinterpret_cast<int32_t*>(given_before + n);
    int32_t* const new_of = len_of + n;
    const int head_in = p.ring_state[0], count = p.ring_state[1];
    if (tid == 0)
        bad_ = 0;
    __syncthreads();

    // each thread has kPer requests side by side; what a bad length would count is cut so that no sum overflows (n_rows < 2^19 + 1, 4096
    // requests: below 2^32)
    int len[kPer], add[kPer];
    Three each[kPer], sum = {0, 0, 0};
    int bad = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
    {
        const int b = tid * kPer + i;
        len[i] = add[i] = 0;
        each[i] = {0, 0, 0};
        if (b < n)
        {
            len[i] = p.lens[b];
            add[i] = p.new_lens[b];
            const int room = p.max_blocks << shift;
            if (len[i] < 0)
                bad |= 8;
            const int held = min(max(len[i], 0), room), grow = min(max(add[i], 0), p.n_rows + 1);
            const int have = (held + (1 << shift) - 1) >> shift;
            int need = have;
            if (add[i] >= 0)
                need = (int) (((int64_t) held + grow + (1 << shift) - 1) >> shift);
            if (len[i] > room || need > p.max_blocks)
            {
                bad |= 1;
                need = min(need, p.max_blocks);
            }
            each[i] = {(uint32_t) grow, (uint32_t) (max(need, have) - have), add[i] < 0 ? (uint32_t) have : 0u};
        }
        sum.a += each[i].a;
        sum.b += each[i].b;
        sum.c += each[i].c;
    }
    const Three incl = wave_scan(sum);
    if (lane == 63)
        wave_sum_[wave] = incl;
    if (bad)
        atomicOr(&bad_, bad);
    __syncthreads();
    Three at = {incl.a - sum.a, incl.b - sum.b, incl.c - sum.c}, total = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
    {
        const Three s = wave_sum_[w];
        if (w < wave)
            at = {at.a + s.a, at.b + s.b, at.c + s.c};
        total = {total.a + s.a, total.b + s.b, total.c + s.c};
    }
    bad = bad_;
    if (total.b > (uint32_t) max(count, 0))
        bad |= 2;
    if (total.a > (uint32_t) p.n_rows)
        bad |= 4;
    if (count < 0 || head_in < 0 || head_in >= p.num_blocks || (uint64_t) max(count, 0) + total.c > (uint64_t) p.num_blocks)
        bad |= 8;
    const bool good = bad == 0;
    const uint32_t blocks = (uint32_t) p.num_blocks;
    const uint32_t head = good ? (uint32_t) head_in : 0u;

    // the state is read above by every thread that needs it, before the barrier; one workgroup at most runs when it is written in place
    const bool first = blockIdx.x == 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
    {
        const int b = tid * kPer + i;
        if (b >= n)
            break;
        rows_before[b] = at.a;
        taken_before[b] = at.b;
        given_before[b] = at.c;
        len_of[b] = len[i];
        new_of[b] = add[i];
        if (first && part != PART_STATE)
            p.cu_tokens[b] = good ? (int32_t) at.a : 0;
        if (first && part != PART_ROWS)
            p.lens_out[b] = !good ? len[i] : add[i] < 0 ? 0 : len[i] + add[i];
        at = {at.a + each[i].a, at.b + each[i].b, at.c + each[i].c};
    }
    if (first && tid == 0)
    {
        if (part != PART_STATE)
        {
            p.cu_tokens[n] = good ? (int32_t) total.a : 0;
            p.status[0] = bad;
        }
        if (part != PART_ROWS)
        {
            p.ring_state_out[0] = good ? (int32_t) ((head + total.b) % blocks) : head_in;
            p.ring_state_out[1] = good ? (int32_t) ((uint32_t) count - total.b + total.c) : count;
        }
    }
    if (part == PART_STATE)
        return;
    if (tid == 0)
        rows_before[n] = total.a;
    __syncthreads();

    // returned pages: behind the ring's end, a wave per ended request.  No other workgroup reads these places of the ring (pages are
    // taken from what the ring held before) or writes these rows of the table.
    if (good && total.c)
        for (int b = blockIdx.x * kWaves + wave; b < n; b += gridDim.x * kWaves)
            if (new_of[b] < 0)
            {
                const int have = (len_of[b] + (1 << shift) - 1) >> shift;
                for (int j = lane; j < have; j += 64)
                    p.ring[(head + (uint32_t) count + given_before[b] + j) % blocks] = p.block_table[(int64_t) b * p.table_stride + j];
            }

    for (int t = blockIdx.x * kThreads + tid; t < p.n_rows; t += gridDim.x * kThreads)
    {
        int slot = -1, pos = -1;
        if (good && (uint32_t) t < total.a)
        {
            int lo = 0, hi = n; // the last request whose rows begin at or before t: rows_before[lo] <= t < rows_before[hi]
            while (hi - lo > 1)
            {
                const int mid = (lo + hi) >> 1;
                if (rows_before[mid] <= (uint32_t) t)
                    lo = mid;
                else
                    hi = mid;
            }
            pos = len_of[lo] + (int) ((uint32_t) t - rows_before[lo]);
            const int page = pos >> shift, off = pos & ((1 << shift) - 1), have = (len_of[lo] + (1 << shift) - 1) >> shift;
            int32_t* const entry = p.block_table + (int64_t) lo * p.table_stride + page;
            int block;
            if (page >= have)
            {
                block = p.ring[(head + taken_before[lo] + (uint32_t) (page - have)) % blocks];
                if (off == 0)
                    *entry = block;
            }
            else
                block = *entry;
            slot = (block << shift) + off;
            if ((uint32_t) block >= blocks)
                slot = -1; // no block of the pool: a ring or table that the caller has not filled
        }
        p.slot_map[t] = slot;
        p.positions[t] = pos;
    }
}
} // namespace

int launch_paged_plan(const tllm_paged_plan_params_t& p, hipStream_t stream)
{
    const int shift = __builtin_ctz((unsigned) p.page_size);
    const size_t lds = ((size_t) 5 * p.n_seqs + 1) * 4;
    launch_util::ensure_dynamic_lds(reinterpret_cast<const void*>(&plan_kernel), lds);
    const int groups = std::max(1, std::min(launch_util::device_cus(), (p.n_rows + kRowsPerGroup - 1) / kRowsPerGroup));
    const bool in_place = p.lens_out == p.lens || p.ring_state_out == p.ring_state;
    if (groups == 1 || !in_place)
        plan_kernel<<<groups, kThreads, lds, stream>>>(p, shift, PART_ALL);
    else
    {
        plan_kernel<<<groups, kThreads, lds, stream>>>(p, shift, PART_ROWS);
        plan_kernel<<<1, kThreads, lds, stream>>>(p, shift, PART_STATE);
    }
    return launched("tllm_paged_plan");
}

} // namespace kernels
} // namespace tllm
