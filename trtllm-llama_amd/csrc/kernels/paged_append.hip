// Keys and values into the 8-bit cache with a scale for each page and head, keys and queries rotated on the way (tllm_paged_append).
//
// A page's scale is shared by all that the page and head hold, so the unit of work is a RUN: the consecutive rows that go to one page.  A
// row begins a run if its slot starts a page or does not follow the slot of the row before it.  One workgroup takes one
// (run, head, key or value): it reads the run's values once into registers, reduces their largest magnitude, settles the scale, brings what the
// page held to it where it grew, and writes 8-bit elements.  Page size * head size / 32 threads, 32 values each, whatever the page:
//   keys    [page][head]: a thread has pairs of 8-element pieces whose elements turn against each other (two 16-byte loads, two
//           8-byte stores);
//   values  [head][page]: a thread has two channels of 16 tokens, one 4-byte load a token, and so one whole 16-byte piece of the page for each
//           channel - the transposition costs nothing, and a piece that is partly new is read, changed and written by its only owner.
// Queries are turned by further workgroups of the same launch.  Bound by bytes for prompts (5500 rows of 32 heads on 8, bfloat16 to e4m3, 126 MB: 32
// us, 3.9 TB/s where a copy reaches 5.0), by the chain slots -> values -> largest -> scale -> store for tokens (64 of them: 8 us; a token touches
// a line of its page for each of its value channels).
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
constexpr int kMaxChunk = 128, kMaxPage = 128;
constexpr float kFloor = 0x1p-100f;

template <bool BF16>
__device__ __forceinline__ float to_f32(uint32_t bits16)
{
    if constexpr (BF16)
        return bf2f((uint16_t) bits16);
    else
        return h2f((uint16_t) bits16);
}

// what enters the cache: infinities (and what rotation brought beyond the type) count as the type's largest value; a NaN stays one
template <bool BF16>
__device__ __forceinline__ float finite(float x)
{
    const float top = BF16 ? 3.38953139e38f : 65504.f;
    return x > top ? top : (x < -top ? -top : x);
}

template <bool FP8>
__device__ __forceinline__ uint32_t four(float a, float b, float c, float d)
{
    if constexpr (FP8)
    {
        a = a != a ? 0.f : a;
        b = b != b ? 0.f : b;
        c = c != c ? 0.f : c;
        d = d != d ? 0.f : d;
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    }
    else
        return (uint32_t) (uint8_t) f2i8_rni_sat(a) | (uint32_t) (uint8_t) f2i8_rni_sat(b) << 8 | (uint32_t) (uint8_t) f2i8_rni_sat(c) << 16
            | (uint32_t) (uint8_t) f2i8_rni_sat(d) << 24;
}

// four held elements under a scale that became 1 / ratio times as large
template <bool FP8>
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float ratio)
{
    if constexpr (FP8)
        return four<true>(__builtin_amdgcn_cvt_f32_fp8((int) w, 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int) w, 1) * ratio,
            __builtin_amdgcn_cvt_f32_fp8((int) w, 2) * ratio, __builtin_amdgcn_cvt_f32_fp8((int) w, 3) * ratio);
    else
        return four<false>((float) (int8_t) w * ratio, (float) (int8_t) (w >> 8) * ratio, (float) (int8_t) (w >> 16) * ratio,
            (float) (int8_t) (w >> 24) * ratio);
}

// product and difference each rounded by themselves: the value does not hang on how the compiler joins them
__device__ __forceinline__ void turn(float& a, float& b, float c, float s)
{
#pragma clang fp contract(off)
    const float x = a * c - b * s, y = b * c + a * s;
    a = x;
    b = y;
}

// The 16 elements of unit u of a row of `dim`: two pieces of 8.  In the rotated part the second piece is what the first turns against (pairs
// i, i + rot / 2) or simply the next one (pairs 2 i, 2 i + 1, and the part that is not rotated).
struct Unit
{
    int lo, hi, turns; // first elements of the pieces; the unit's first angle, or -1
};
__device__ __forceinline__ Unit unit_at(int u, int rot, bool pairs)
{
    if (u * 16 >= rot)
        return {u * 16, u * 16 + 8, -1};
    return pairs ? Unit{u * 16, u * 16 + 8, u * 8} : Unit{u * 8, u * 8 + (rot >> 1), u * 8};
}

template <bool BF16>
__device__ __forceinline__ void load_unit(float (&x)[16], const uint16_t* row, const Unit& u, const float* rope, int rot, int pos, bool pairs)
{
    const uint4 a = *reinterpret_cast<const uint4*>(row + u.lo), b = *reinterpret_cast<const uint4*>(row + u.hi);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        x[2 * i] = to_f32<BF16>(w[i] & 0xffffu);
        x[2 * i + 1] = to_f32<BF16>(w[i] >> 16);
    }
    if (u.turns < 0)
        return;
    const float4* at = reinterpret_cast<const float4*>(rope + ((int64_t) pos * (rot >> 1) + u.turns) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const float4 r = at[i]; // two angles
        if (pairs)
        {
            turn(x[4 * i], x[4 * i + 1], r.x, r.y);
            turn(x[4 * i + 2], x[4 * i + 3], r.z, r.w);
        }
        else
        {
            turn(x[2 * i], x[2 * i + 8], r.x, r.y);
            turn(x[2 * i + 1], x[2 * i + 9], r.z, r.w);
        }
    }
}

// The slot of row t and its place in the rope table; what is no place of the pool, or has no angle, has slot -1.
struct Row
{
    int slot, place;
};
__device__ __forceinline__ Row row_at(const tllm_paged_append_params_t& p, int t, int shift)
{
    Row r = {-1, 0};
    if (t >= 0 && t < p.n_rows)
    {
        r.slot = p.slot_map[t];
        if (p.rot_dim)
            r.place = p.positions[t];
        if ((uint32_t) r.slot >= (uint32_t) p.num_blocks << shift || (p.rot_dim && (uint32_t) r.place >= (uint32_t) p.rope_len))
            r.slot = -1;
    }
    return r;
}

__device__ __forceinline__ bool begins(int slot, int before, int page) // a run
{
    return slot >= 0 && !(before >= 0 && before + 1 == slot && (slot & (page - 1)) != 0);
}

template <int DIM, bool BF16, bool FP8>
__global__ __launch_bounds__(DIM * kMaxPage / 32) void append_kernel(const tllm_paged_append_params_t p, const int shift, const int chunk)
{
    __shared__ int slots[kMaxChunk + kMaxPage + 1], places[kMaxChunk + kMaxPage + 1];
    __shared__ float red[32];
    const int page = 1 << shift, t0 = blockIdx.x * chunk, tid = threadIdx.x;
    const int kv_jobs = 2 * p.kv_heads;
    const bool pairs = p.rope_pairs != 0;
    if ((int) blockIdx.y < kv_jobs)
    {
        // most chunks of a prompt have no run's beginning: every wave sees that by itself
        bool any = false;
        for (int i = 0; i < chunk && !any; i += 63)
        {
            const int here = i + (tid & 63) - 1, slot = here < chunk ? row_at(p, t0 + here, shift).slot : -1;
            const int before = __shfl_up(slot, 1, 64);
            any = __builtin_amdgcn_ballot_w64((tid & 63) > 0 && begins(slot, before, page)) != 0;
        }
        if (!any)
            return;
    }
    for (int i = tid; i < chunk + page + 1; i += blockDim.x) // the row before the chunk, the chunk, and as many behind it as a run can go on for
    {
        const Row at = row_at(p, t0 - 1 + i, shift);
        slots[i] = at.slot;
        places[i] = at.place;
    }
    __syncthreads();

    if ((int) blockIdx.y >= kv_jobs) // queries: a unit a thread
    {
        constexpr int kUnits = DIM / 16;
        const int per_row = p.q_heads * kUnits, u = (blockIdx.y - kv_jobs) * blockDim.x + tid;
        const int r = u / per_row, t = t0 + r;
        if (r >= chunk || t >= p.n_rows || slots[1 + r] < 0)
            return;
        const int hu = u - r * per_row, h = hu / kUnits;
        const Unit at = unit_at(hu - h * kUnits, p.rot_dim, pairs);
        float x[16];
        load_unit<BF16>(x, static_cast<const uint16_t*>(p.q) + t * p.q_row + h * p.q_head, at, p.rope, p.rot_dim, places[1 + r], pairs);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = BF16 ? (uint32_t) f2bf(x[2 * i]) | (uint32_t) f2bf(x[2 * i + 1]) << 16 : (uint32_t) f2h(x[2 * i]) | (uint32_t) f2h(x[2 * i + 1]) << 16;
        uint16_t* const to = static_cast<uint16_t*>(p.q_out) + t * p.q_out_row + h * p.q_out_head;
        *reinterpret_cast<uint4*>(to + at.lo) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(to + at.hi) = make_uint4(w[4], w[5], w[6], w[7]);
        return;
    }

    constexpr float top = FP8 ? 448.f : 127.f;
    const int head = blockIdx.y >> 1, which = blockIdx.y & 1, lane = tid & 63;
    const int threads = page * DIM / 32; // the last wave of a small page may be half empty
    for (int r = 0; r < chunk; ++r)
    {
        const int s0 = __builtin_amdgcn_readfirstlane(slots[1 + r]), before = __builtin_amdgcn_readfirstlane(slots[r]);
        const int off = s0 & (page - 1);
        if (!begins(s0, before, page))
            continue; // nothing, or the middle of a run
        int n = 0; // rows of the run
        for (int j0 = 0; j0 < page - off; j0 += 64)
        {
            const int j = j0 + lane;
            const uint64_t mine = __builtin_amdgcn_ballot_w64(j < page - off && slots[1 + r + min(j, page)] == s0 + j);
            n += ~mine ? __builtin_ctzll(~mine) : 64;
            if (~mine)
                break;
        }
        const int t = t0 + r;
        const int64_t block = s0 >> shift;
        uint8_t* const base = static_cast<uint8_t*>(p.pool) + ((block * 2 + which) * p.kv_heads + head) * (int64_t) (page * DIM);
        float* const scale_at = p.scales + (block * 2 + which) * p.kv_heads + head;
        const float old = off ? *scale_at : 0.f;

        // everything that is read of memory is sent for here, before the first of it is waited for
        float x[32];
        float big = kFloor;
        uint4 was[2] = {}; // the thread's two pieces of a page of values, where they are not wholly new
        const int v_first = tid / (DIM / 2) * 16, lo = off - v_first, hi = off + n - v_first; // of its 16 places those in [lo, hi) are new, those before held
        uint4* const v_at = reinterpret_cast<uint4*>(base + tid % (DIM / 2) * 2 * page + v_first);
        const bool partly = which == 1 && tid < threads && hi > 0 && (lo > 0 || hi < 16);
        if (partly)
        {
            was[0] = *v_at;
            was[1] = v_at[page / 16];
        }
        if (which == 0)
        {
            constexpr int kUnits = DIM / 16;
            const int u = tid % kUnits, step = threads / kUnits; // step = page / 2 rows at a time
            const Unit at = unit_at(u, p.rot_dim, pairs);
#pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                const int row = tid / kUnits + half * step;
                float y[16] = {};
                if (tid < threads && row < n)
                    load_unit<BF16>(y, static_cast<const uint16_t*>(p.k) + (t + row) * p.k_row + head * p.k_head, at, p.rope, p.rot_dim,
                        places[1 + r + row], pairs);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    x[half * 16 + i] = finite<BF16>(y[i]);
            }
        }
        else
        {
            constexpr int kPairs = DIM / 2;
            const int d = tid % kPairs * 2, g = tid / kPairs * 16 - off; // the thread's tokens are rows g .. g + 15 of the run
            const uint16_t* const from = static_cast<const uint16_t*>(p.v) + head * p.v_head + d;
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                uint32_t w = 0;
                if (tid < threads && g + i >= 0 && g + i < n)
                    w = *reinterpret_cast<const uint32_t*>(from + (t + g + i) * p.v_row);
                x[i] = finite<BF16>(to_f32<BF16>(w & 0xffffu));
                x[16 + i] = finite<BF16>(to_f32<BF16>(w >> 16));
            }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i)
            big = fmaxf(big, fabsf(x[i])); // a NaN does not count
        big = block_max(big, red);
        const float scale = fmaxf(old, big / top), ratio = old / scale;
        const bool grew = off && scale > old;
        if (tid == 0 && (grew || !off))
            *scale_at = scale;
        if (which == 0)
        {
            constexpr int kUnits = DIM / 16;
            const int u = tid % kUnits, step = threads / kUnits;
            const Unit at = unit_at(u, p.rot_dim, pairs);
#pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                const int row = tid / kUnits + half * step;
                if (tid < threads && row < n)
                {
                    uint8_t* const to = base + (off + row) * DIM;
                    const float* const y = x + half * 16;
                    *reinterpret_cast<uint2*>(to + at.lo)
                        = make_uint2(four<FP8>(y[0] / scale, y[1] / scale, y[2] / scale, y[3] / scale), four<FP8>(y[4] / scale, y[5] / scale, y[6] / scale, y[7] / scale));
                    *reinterpret_cast<uint2*>(to + at.hi)
                        = make_uint2(four<FP8>(y[8] / scale, y[9] / scale, y[10] / scale, y[11] / scale), four<FP8>(y[12] / scale, y[13] / scale, y[14] / scale, y[15] / scale));
                }
            }
            if (grew)
                for (int i = tid * 16; i < off * DIM; i += blockDim.x * 16)
                {
                    uint4 w = *reinterpret_cast<const uint4*>(base + i);
                    w = make_uint4(rescaled<FP8>(w.x, ratio), rescaled<FP8>(w.y, ratio), rescaled<FP8>(w.z, ratio), rescaled<FP8>(w.w, ratio));
                    *reinterpret_cast<uint4*>(base + i) = w;
                }
        }
        else if (tid < threads)
        {
            if (n == 1 && !grew) // a token by itself: a byte a channel
            {
                if (lo >= 0 && lo < 16)
                {
                    float one[2] = {};
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (i == lo)
                            one[0] = x[i], one[1] = x[16 + i];
                    const uint32_t w = four<FP8>(one[0] / scale, one[1] / scale, 0.f, 0.f);
                    reinterpret_cast<uint8_t*>(v_at)[lo] = (uint8_t) w;
                    reinterpret_cast<uint8_t*>(v_at)[page + lo] = (uint8_t) (w >> 8);
                }
            }
            else if (hi > 0 && (lo < 16 || grew))
#pragma unroll
                for (int c = 0; c < 2; ++c)
                {
                    uint32_t w[4] = {was[c].x, was[c].y, was[c].z, was[c].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                    {
                        const float* const y = x + c * 16 + i * 4;
                        const uint32_t held = grew ? rescaled<FP8>(w[i], ratio) : w[i];
                        const uint32_t fresh = four<FP8>(y[0] / scale, y[1] / scale, y[2] / scale, y[3] / scale);
                        uint32_t out = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                        {
                            const uint32_t byte = 0xffu << (8 * e);
                            const int at = i * 4 + e;
                            out |= (at < lo ? held : at < hi ? fresh : w[i]) & byte;
                        }
                        w[i] = out;
                    }
                    v_at[c * (page / 16)] = make_uint4(w[0], w[1], w[2], w[3]);
                }
        }
        r += n - 1;
    }
}

template <int DIM, bool BF16>
void launch_dim(const tllm_paged_append_params_t& p, hipStream_t stream)
{
    const int shift = __builtin_ctz((unsigned) p.page_size), threads = std::max(64, p.page_size * DIM / 32);
    // Rows a workgroup looks for runs in.  The host does not know whether they are tokens (a run each, that want workgroups of their own) or
    // prompts (a run a page, where workgroups without one are most of the time): one row while that makes few workgroups, up to 16 where the
    // chip is full of them either way, a page where that leaves thousands (us at 1 / 8 / 16 / 64 rows, 8 heads of 128: 64 tokens 8 / 25 / 44 / 168,
    // 512 tokens 42 / 34 / 52 / 178, a prompt of 1024 74 / 26 / 18 / 12, prompts of 5459 82 / 32 / 34 / 32).  Rows times heads are taken for a prompt, and
    // tokens that make as many pay for it, a run behind the other: 64 tokens of 32 heads 19 us, 128 34, 1024 255 (a prompt of as many 23), 64 beside a
    // prompt of 1024 190.
    const int64_t work = (int64_t) p.n_rows * p.kv_heads;
    int chunk = 1;
    while (chunk * 2 <= std::min(16, p.page_size) && chunk * 2 * 512 <= work)
        chunk *= 2;
    if (work >= 32768)
        chunk = p.page_size;
    const int q_groups = p.q_heads ? (chunk * p.q_heads * (DIM / 16) + threads - 1) / threads : 0;
    const dim3 grid((p.n_rows + chunk - 1) / chunk, 2 * p.kv_heads + q_groups);
    if (p.cache_type == TLLM_FP8)
        append_kernel<DIM, BF16, true><<<grid, threads, 0, stream>>>(p, shift, chunk);
    else
        append_kernel<DIM, BF16, false><<<grid, threads, 0, stream>>>(p, shift, chunk);
}
} // namespace

int launch_paged_append(const tllm_paged_append_params_t& p, hipStream_t stream)
{
    const bool bf16 = p.dtype == TLLM_BF16;
    switch (p.head_size)
    {
    case 64: bf16 ? launch_dim<64, true>(p, stream) : launch_dim<64, false>(p, stream); break;
    case 128: bf16 ? launch_dim<128, true>(p, stream) : launch_dim<128, false>(p, stream); break;
    default: bf16 ? launch_dim<256, true>(p, stream) : launch_dim<256, false>(p, stream); break;
    }
    return launched("tllm_paged_append");
}

} // namespace kernels
} // namespace tllm
