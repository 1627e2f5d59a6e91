// Attention over the 8-bit cache with a scale for each page and head (tllm_paged_attention).
//
// rows_kernel: one workgroup per (request, key head, 16 rows, part of the keys).  The rows of a key head are its query heads of one token,
// then those of the next, so that a decoded token of grouped heads is one tile.  Four waves take tiles of 64 keys in turn; each runs the
// one-pass softmax (running maximum m and sum l, O rescaled when m grows) and they join through LDS.
//   S^T = K Q^T by v_mfma_f32_16x16x32_f16, O^T += V^T P^T by the same.  Which key an MFMA row stands for, and which dimension or key a
//   k-element, is free as long as both operands agree, so it is chosen for the cache's bytes: lane l = 16 g + r of tile t takes key
//   16 (r / 4) + 4 t + r % 4, whose scores come back to the lanes of group g = r / 4 of the result, 16 consecutive keys a lane; of a
//   key a lane takes dimensions 64 j + 16 g .. + 15 (two k-steps).  Every load is 16 bytes of a row of keys or of a channel of values,
//   no operand passes through LDS, and P goes from the first product's registers into the second's as it is.
//   16 keys lie in one page, so a lane has one key scale and one value scale per tile.
// 8-bit elements become fp16 exactly (int8: 0x6400 | (q + 128) = 1152 + q; e4m3: the convert instruction); scales enter in fp32: the key's with the
// softmax scale behind the first product, the value's into P relative to the largest value scale so far, times 2^15 (P <= 1 and the
// ratio <= 1: nothing overflows, and nothing is lost until a page's scale is 2^-29 of another's).
// Few rows and long contexts: the keys are also split over workgroups, the parts joined by merge_kernel in fp32.
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
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kPScale = 32768.f; // 2^15, see above
constexpr int kTile = 64;

__device__ __forceinline__ f16x8 join(u32x4 w)
{
    return __builtin_bit_cast(f16x8, w);
}

// 8 bytes -> 8 fp16
template <bool FP8>
__device__ __forceinline__ f16x8 eight(uint32_t a, uint32_t b)
{
    u32x4 o;
    if constexpr (FP8)
    {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true));
    }
    else
    {
        const h2_t bias = {(_Float16) 1152.f, (_Float16) 1152.f};
        const uint32_t magic = 0x64646464u;
        a ^= 0x80808080u;
        b ^= 0x80808080u;
        o[0] = h2_as_u32(u32_as_h2(__builtin_amdgcn_perm(magic, a, 0x04010400u)) - bias);
        o[1] = h2_as_u32(u32_as_h2(__builtin_amdgcn_perm(magic, a, 0x04030402u)) - bias);
        o[2] = h2_as_u32(u32_as_h2(__builtin_amdgcn_perm(magic, b, 0x04010400u)) - bias);
        o[3] = h2_as_u32(u32_as_h2(__builtin_amdgcn_perm(magic, b, 0x04030402u)) - bias);
    }
    return join(o);
}

__device__ __forceinline__ float groups_max(float v) // over the four lanes of one result column
{
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float groups_sum(float v)
{
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) // to nearest
{
    f16x2 r = {(_Float16) a, (_Float16) b};
    return __builtin_bit_cast(uint32_t, r);
}

// one request's part of the batch, cut to what the buffers hold
struct Request
{
    int row0, rows, len;
};
__device__ __forceinline__ Request request_of(const tllm_paged_attention_params_t& p, int b, int shift)
{
    Request r;
    r.row0 = p.cu_tokens[b];
    r.rows = p.cu_tokens[b + 1] - r.row0;
    if (r.row0 < 0 || r.rows < 0 || r.rows > p.n_rows - r.row0)
        r.rows = 0;
    r.len = min(max(p.kv_lens[b], 0), p.max_blocks << shift);
    return r;
}

// Fragments of a query row: k-steps 2 j and 2 j + 1 of a lane are dimensions 64 j + 16 g .. + 15.  A bfloat16 row is taken to fp16 under a power
// of two that brings its largest value to [1, 2); returns what the scores have to be multiplied by.
template <int DIM, bool BF16>
__device__ __forceinline__ float load_query(f16x8 (&q)[DIM / 32], const uint16_t* row, int g)
{
    u32x4 w[DIM / 32];
#pragma unroll
    for (int j = 0; j < DIM / 64; ++j)
    {
        const uint4* at = reinterpret_cast<const uint4*>(row + 64 * j + 16 * g);
        const uint4 a = row ? at[0] : make_uint4(0, 0, 0, 0), b = row ? at[1] : make_uint4(0, 0, 0, 0);
        w[2 * j] = u32x4{a.x, a.y, a.z, a.w};
        w[2 * j + 1] = u32x4{b.x, b.y, b.z, b.w};
    }
    float back = 1.f;
    if constexpr (BF16)
    {
        uint32_t top = 0; // magnitudes compare as integers
#pragma unroll
        for (int s = 0; s < DIM / 32; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                top = max(top, max(w[s][i] & 0x7fffu, (w[s][i] >> 16) & 0x7fffu));
        top = max(top, (uint32_t) __shfl_xor((int) top, 16, 64));
        top = max(top, (uint32_t) __shfl_xor((int) top, 32, 64));
        const int e = max(1, min(253, (int) (top >> 7))); // a row of zeros or subnormals: 2^126 times, of infinities: they stay infinite
        const float to = __builtin_bit_cast(float, (uint32_t) (254 - e) << 23);
        back = __builtin_bit_cast(float, (uint32_t) e << 23);
#pragma unroll
        for (int s = 0; s < DIM / 32; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[s][i] = pack_f16(bf2f((uint16_t) w[s][i]) * to, bf2f((uint16_t) (w[s][i] >> 16)) * to);
    }
#pragma unroll
    for (int s = 0; s < DIM / 32; ++s)
        q[s] = join(w[s]);
    return back;
}

// bytes of `w` (keys first .. first + 15) from key `end` on become 0: what a page holds behind its last token is anything, and 0 times a NaN is one
__device__ __forceinline__ u32x4 cut(u32x4 w, int keep)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const int n = keep - 4 * i; // bytes of the word that stay
        w[i] = n >= 4 ? w[i] : n <= 0 ? 0u : w[i] & (0xffffffffu >> (32 - 8 * n));
    }
    return w;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_out(float a, float b)
{
    if constexpr (BF16)
        return (uint32_t) f2bf(a) | (uint32_t) f2bf(b) << 16;
    else
        return (uint32_t) f2h(a) | (uint32_t) f2h(b) << 16;
}

struct Split
{
    float* o;  // [n_rows][q_heads][parts][DIM], not divided by l
    float* ml; // [n_rows][q_heads][parts][2]
    int parts;
};

template <int DIM, bool BF16, bool FP8>
__global__ __launch_bounds__(256) void rows_kernel(const tllm_paged_attention_params_t p, const int shift, const int row_tiles, const Split split)
{
    constexpr int kSteps = DIM / 32, kOut = DIM / 16, kLine = DIM + 4;
    __shared__ float acc[2][16][kLine];
    __shared__ float ms[4][16], ls[4][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    int id = blockIdx.x;
    const int part = id % split.parts;
    id /= split.parts;
    const int tile = id % row_tiles;
    id /= row_tiles;
    const int head = id % p.kv_heads, b = id / p.kv_heads, group = p.q_heads / p.kv_heads;
    const Request req = request_of(p, b, shift);
    const int rows = min(req.rows, p.max_new) * group, row = tile * 16 + r;
    if (tile * 16 >= rows)
        return;
    const int first = req.len - req.rows; // position of the request's first row
    const bool live = row < rows;
    const int token = row / group, qh = head * group + row - token * group;
    const int seen = live ? first + token + 1 : 0; // keys [from, seen) are visible to the lane's row
    const int from = p.window > 0 ? seen - p.window : 0;
    const int last = min(tile * 16 + 15, rows - 1) / group;
    const int lo = p.window > 0 ? max(0, first + tile * 16 / group + 1 - p.window) : 0, hi = first + last + 1;
    const int t_lo = lo / kTile, n_tiles = max(0, (hi + kTile - 1) / kTile - t_lo), per = (n_tiles + split.parts - 1) / split.parts;
    const int t_begin = t_lo + min(n_tiles, part * per), t_end = t_lo + min(n_tiles, (part + 1) * per);

    f16x8 q[kSteps];
    const uint16_t* const q_row = live ? static_cast<const uint16_t*>(p.q) + (req.row0 + token) * p.q_row + qh * p.q_head : nullptr;
    const float factor = load_query<DIM, BF16>(q, q_row, g) * p.scale * kLog2e;

    const int page = 1 << shift;
    const int64_t head_bytes = (int64_t) page * DIM, side_bytes = head_bytes * p.kv_heads;
    const uint8_t* const pool = static_cast<const uint8_t*>(p.pool) + head * head_bytes;
    const int32_t* const table = p.block_table + (int64_t) b * p.table_stride;

    f32x4 o[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i)
        o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f, v_ref = 0.f;
    for (int t = t_begin + wave; t < t_end; t += 4)
    {
        const int key0 = t * kTile;
        const int kk = key0 + 16 * (r >> 2), vk = key0 + 16 * g; // first keys of the lane's 16 in the first and the second product
        const int kb = kk < req.len ? table[kk >> shift] : -1, vb = vk < req.len ? table[vk >> shift] : -1;
        const bool k_in = (uint32_t) kb < (uint32_t) p.num_blocks, v_in = (uint32_t) vb < (uint32_t) p.num_blocks;
        const uint8_t* const k_at = pool + (int64_t) (k_in ? kb : 0) * 2 * side_bytes + ((kk & (page - 1)) + (r & 3)) * DIM + 16 * g;
        const uint8_t* const v_at = pool + ((int64_t) (v_in ? vb : 0) * 2 + 1) * side_bytes + r * page + (vk & (page - 1));
        const float* const s_at = p.scales + (int64_t) (v_in ? vb : 0) * 2 * p.kv_heads + head;
        const float ks = v_in ? s_at[0] : 0.f, vs = v_in ? s_at[p.kv_heads] : 0.f;

        float s[16];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < DIM / 64; ++j)
            {
                const u32x4 w = *reinterpret_cast<const u32x4*>(k_at + 4 * i * DIM + 64 * j);
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(w[0], w[1]), q[2 * j], c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(w[2], w[3]), q[2 * j + 1], c, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[4 * i + e] = c[e];
        }
        const float f = factor * ks;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            const int key = vk + i;
            s[i] = v_in && key < seen && key >= from ? s[i] * f : -INFINITY;
            top = fmaxf(top, s[i]);
        }
        const float m_new = fmaxf(m, groups_max(top)), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float v_new = fmaxf(v_ref, groups_max(vs));
        const float alpha = __builtin_amdgcn_exp2f(m - m_use);
        if (__builtin_amdgcn_ballot_w64(m_new != m || v_new != v_ref))
        {
            const float back = alpha * (v_new > 0.f ? v_ref / v_new : 1.f);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < kOut; ++i)
                o[i] *= back;
        }
        m = m_new;
        v_ref = v_new;
        const float up = v_new > 0.f ? vs / v_new * kPScale : 0.f;
        u32x4 w[2];
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const float a = __builtin_amdgcn_exp2f(s[2 * i] - m_use), c = __builtin_amdgcn_exp2f(s[2 * i + 1] - m_use);
            l += a + c;
            w[i >> 2][i & 3] = pack_f16(a * up, c * up);
        }
        const f16x8 p0 = join(w[0]), p1 = join(w[1]);
        const int keep = v_in ? req.len - vk : 0;
        const bool whole = __builtin_amdgcn_ballot_w64(keep < 16) == 0;
#pragma unroll
        for (int i = 0; i < kOut; ++i)
        {
            u32x4 v = *reinterpret_cast<const u32x4*>(v_at + 16 * i * page);
            if (!whole)
                v = cut(v, keep);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(v[0], v[1]), p0, o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(v[2], v[3]), p1, o[i], 0, 0, 0);
        }
    }

    // the waves' parts -> one
    l = groups_sum(l);
    if (g == 0)
    {
        ms[wave][r] = m;
        ls[wave][r] = l;
    }
    __syncthreads();
    const float m_all = fmaxf(fmaxf(ms[0][r], ms[1][r]), fmaxf(ms[2][r], ms[3][r])), m_use = m_all == -INFINITY ? 0.f : m_all;
    const float mine = __builtin_amdgcn_exp2f(m - m_use) * (v_ref * (1.f / kPScale));
    if (wave >= 2)
#pragma unroll
        for (int i = 0; i < kOut; ++i)
            *reinterpret_cast<f32x4*>(&acc[wave - 2][r][16 * i + 4 * g]) = o[i] * mine;
    __syncthreads();
    if (wave < 2)
#pragma unroll
        for (int i = 0; i < kOut; ++i)
        {
            f32x4* const at = reinterpret_cast<f32x4*>(&acc[wave][r][16 * i + 4 * g]);
            *at = *at + o[i] * mine;
        }
    __syncthreads();
    for (int u = tid; u < 16 * DIM / 8; u += 256)
    {
        const int ur = u / (DIM / 8), d = u % (DIM / 8) * 8, urow = tile * 16 + ur;
        if (urow >= rows)
            continue;
        const float um = fmaxf(fmaxf(ms[0][ur], ms[1][ur]), fmaxf(ms[2][ur], ms[3][ur])), uu = um == -INFINITY ? 0.f : um;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            sum += ls[w][ur] * __builtin_amdgcn_exp2f(ms[w][ur] - uu);
        const f32x4 a = *reinterpret_cast<const f32x4*>(&acc[0][ur][d]) + *reinterpret_cast<const f32x4*>(&acc[1][ur][d]);
        const f32x4 c = *reinterpret_cast<const f32x4*>(&acc[0][ur][d + 4]) + *reinterpret_cast<const f32x4*>(&acc[1][ur][d + 4]);
        const int utoken = urow / group, uh = head * group + urow - utoken * group;
        if (split.parts > 1)
        {
            const int64_t at = ((int64_t) (req.row0 + utoken) * p.q_heads + uh) * split.parts + part;
            *reinterpret_cast<f32x4*>(split.o + at * DIM + d) = a;
            *reinterpret_cast<f32x4*>(split.o + at * DIM + d + 4) = c;
            if (d == 0)
            {
                split.ml[2 * at] = um;
                split.ml[2 * at + 1] = sum;
            }
            continue;
        }
        const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum); // a row that saw nothing is 0, a NaN stays one
        uint16_t* const to = static_cast<uint16_t*>(p.out) + (req.row0 + utoken) * p.out_row + uh * p.out_head + d;
        *reinterpret_cast<uint4*>(to) = make_uint4(pack_out<BF16>(a[0] * inv, a[1] * inv), pack_out<BF16>(a[2] * inv, a[3] * inv),
            pack_out<BF16>(c[0] * inv, c[1] * inv), pack_out<BF16>(c[2] * inv, c[3] * inv));
    }
}

// parts of the keys -> rows: a wave per row and head
template <int DIM, bool BF16>
__global__ __launch_bounds__(256) void merge_kernel(const tllm_paged_attention_params_t p, const int shift, const Split split)
{
    constexpr int kPer = DIM / 64;
    const int lane = threadIdx.x & 63;
    int64_t id = (int64_t) blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int) (id % p.q_heads);
    id /= p.q_heads;
    const int i = (int) (id % p.max_new), b = (int) (id / p.max_new);
    if (b >= p.n_seqs)
        return;
    const Request req = request_of(p, b, shift);
    if (i >= req.rows)
        return;
    const int64_t at = ((int64_t) (req.row0 + i) * p.q_heads + h) * split.parts;
    float m = -INFINITY;
    for (int s = 0; s < split.parts; ++s)
        m = fmaxf(m, split.ml[2 * (at + s)]);
    const float m_use = m == -INFINITY ? 0.f : m;
    float sum = 0.f, o[kPer] = {};
    for (int s = 0; s < split.parts; ++s)
    {
        const float w = __builtin_amdgcn_exp2f(split.ml[2 * (at + s)] - m_use);
        sum += w * split.ml[2 * (at + s) + 1];
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            o[e] += w * split.o[(at + s) * DIM + lane * kPer + e];
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    uint16_t* const to = static_cast<uint16_t*>(p.out) + (req.row0 + i) * p.out_row + h * p.out_head + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
        to[e] = BF16 ? f2bf(o[e] * inv) : f2h(o[e] * inv);
}

// Workgroups that the keys are split into: as many as fill the chip twice over, a part no shorter than 512 keys.
int parts_of(const tllm_paged_attention_params_t& p)
{
    const int row_tiles = ((int64_t) p.max_new * (p.q_heads / p.kv_heads) + 15) / 16;
    if (row_tiles > 1)
        return 1;
    const int64_t groups = (int64_t) p.n_seqs * p.kv_heads;
    const int64_t keys = p.window > 0 ? std::min(p.window, p.max_kv) : p.max_kv;
    const int64_t want = 2 * launch_util::device_cus() / groups, most = keys / 512;
    return (int) std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 64));
}

template <int DIM, bool BF16>
void launch_dim(const tllm_paged_attention_params_t& p, void* workspace, hipStream_t stream)
{
    const int shift = __builtin_ctz((unsigned) p.page_size), parts = parts_of(p);
    const int row_tiles = (int) (((int64_t) p.max_new * (p.q_heads / p.kv_heads) + 15) / 16);
    Split split = {static_cast<float*>(workspace), nullptr, parts};
    if (parts > 1)
        split.ml = split.o + (int64_t) p.n_rows * p.q_heads * parts * DIM;
    const int64_t grid = (int64_t) p.n_seqs * p.kv_heads * row_tiles * parts;
    if (p.cache_type == TLLM_FP8)
        rows_kernel<DIM, BF16, true><<<(unsigned) grid, 256, 0, stream>>>(p, shift, row_tiles, split);
    else
        rows_kernel<DIM, BF16, false><<<(unsigned) grid, 256, 0, stream>>>(p, shift, row_tiles, split);
    if (parts > 1)
        merge_kernel<DIM, BF16><<<(unsigned) (((int64_t) p.n_seqs * p.max_new * p.q_heads + 3) / 4), 256, 0, stream>>>(p, shift, split);
}
} // namespace

size_t paged_attention_workspace(const tllm_paged_attention_params_t& p)
{
    const int parts = parts_of(p);
    return parts > 1 ? (size_t) p.n_rows * p.q_heads * parts * (p.head_size + 2) * 4 : 0;
}

int launch_paged_attention(const tllm_paged_attention_params_t& p, void* workspace, hipStream_t stream)
{
    const bool bf16 = p.dtype == TLLM_BF16;
    switch (p.head_size)
    {
    case 64: bf16 ? launch_dim<64, true>(p, workspace, stream) : launch_dim<64, false>(p, workspace, stream); break;
    case 128: bf16 ? launch_dim<128, true>(p, workspace, stream) : launch_dim<128, false>(p, workspace, stream); break;
    default: bf16 ? launch_dim<256, true>(p, workspace, stream) : launch_dim<256, false>(p, workspace, stream); break;
    }
    return launched("tllm_paged_attention");
}

} // namespace kernels
} // namespace tllm
