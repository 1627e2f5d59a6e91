// Attention over the 8-bit cache with a scale for each page and head (tllm_paged_attention).
//
// The rows of a key head are its query heads of one token, then those of the next, so that a decoded token of grouped heads is one tile of 16 rows.
// Both kernels run the one-pass softmax (running maximum m and sum l, O rescaled when m grows) over tiles of 64 keys:
//   S^T = K Q^T by v_mfma_f32_16x16x32_f16, O^T += V^T P^T by the same.  Which key an MFMA row stands for, and which dimension or key a
//   k-element, is free as long as both operands agree, so it is chosen for the cache's bytes: lane l = 16 g + r of part i takes key
//   16 (r / 4) + 4 i + r % 4, whose scores come back to the lanes of group g = r / 4 of the result, 16 consecutive keys a lane; of a
//   key a lane takes dimensions 64 j + 16 g .. + 15 (two k-steps).  Every load is 16 bytes of a row of keys or of a channel of values, and
//   P goes from the first product's registers into the second's as it is.  16 keys lie in one page, so a lane has one key scale and one value
//   scale per tile.
// 8-bit elements become fp16 exactly (int8: 0x6400 | (q + 128) = 1152 + q; e4m3: the convert instruction).  Scales enter in fp32: the key's with the
// softmax scale behind the first product; the value's in the exponent of the weight, which is 2^7 times exp2(score) * scale over the largest such
// product that the ROW has seen (its logarithm is mv, next to m for the sum).  What a row does not see, and what it does not weigh, does not enter its
// mv: a page with values of 1e38 behind a row or outside its window costs the row nothing.  m and mv are brought along only when something is more
// than 8 (a factor of 2^8) above them: a weight is at most 2^15, nothing overflows, it keeps its 11 bits until it is 2^-21 of the row's largest (where
// 8-bit elements of the largest one's page are half a step, 2^-8 or 2^-10, off), and in most tiles no lane asks another for anything.
//   rows_body   16 rows: four or eight waves take tiles in turn, straight from memory into registers, and join through LDS.  Single tokens are bound by the
//               cache's bytes (48 requests over 4000 to 8000 keys, 8 key heads of 128, e4m3: 111 us, 5.4 TB/s); the keys are also split over workgroups,
//               whose parts merge_kernel joins (131072 keys of one request: 42 + 4 us; a token over 1032, 32 heads: 7 + 4, the chain table -> keys ->
//               softmax -> join).
//   tile_kernel 64 or 128 rows: the waves share the tiles, which they bring to LDS as fp16 fragments, the next one while this one is computed.  Prompts
//               are bound by the arithmetic - products, exponentials, and the conversions, which are once a workgroup here and not once a wave: 0.90
//               PFLOP/s where workgroups fill the chip evenly (2048 tokens behind 20000, 32 heads of 128), 0.64 where 640 of them have 512 places (three
//               prompts of up to 1024 behind up to 2500: 178 us).
#include "dev_utils.h"
#include "launch_util.h"
#include "serving_kernels.h"
#include <algorithm>
#include <type_traits>

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
constexpr float kPShift = 7.f, kSlack = 8.f; // see above
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

// The keys of a row in parts, each by its own workgroup.
struct Split
{
    float* o;     // [rows][q_heads][parts][DIM], not divided by l
    float4* seen; // [rows][q_heads][parts]: m, l, mv
    int parts;
    int per; // rows a request has in these, 0: they are the batch's rows
    __device__ __forceinline__ int64_t at(int b, int row0, int i, int heads, int h) const { return ((int64_t) ((per ? b * per : row0) + i) * heads + h) * parts; }
};

// What a row has seen: m, the largest score; mv, the largest score + log2 of its page's value scale; l, the sum of exp2(score - m).  O is in units of
// exp2(mv - kPShift) until it is stored as the result: what l times the largest bfloat16 value is has no place in fp32.
struct Seen
{
    float m = -INFINITY, mv = -INFINITY, l = 0.f;
};
__device__ __forceinline__ float part_of(float mine, float all) // exp2(mine - all), where a part or all of them may have seen nothing
{
    return all == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - all);
}
__device__ __forceinline__ float result_of(float m, float mv, float l) // of O; a row that saw nothing is 0, a NaN stays one
{
    return (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) * (part_of(mv, m) * __builtin_amdgcn_exp2f(-kPShift));
}

// One tile of one row: the 16 scores of a lane (keys key0 .. + 15 of a query's row), under the key scale `ks` of their page and log2 of its value scale `lv` -> its weights in fp16, with what
// the row has seen and O brought along.  `plain` (the same for the wave): every key is seen.
template <int N>
__device__ __forceinline__ void soften(float (&s)[16], f16x8 (&w)[2], Seen& r, f32x4 (&o)[N], float ks, float lv, float factor, bool plain, bool in, int key0, int from, int seen)
{
    // zero keys under the largest scale score 0, not 0 times an infinity, and masked ones -INFINITY, not 0 times that
    const float f = fminf(fmaxf(factor * ks, 1.17549435e-38f), 3.4028235e38f);
    if (!plain)
    {
        const int begin = from - key0, end = in ? seen - key0 : -1;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[i] = i < end && i >= begin ? s[i] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i)
        top = fmaxf(top, s[i]);
    top *= f; // f > 0
    const float top_v = top + lv;
    if (__builtin_amdgcn_ballot_w64(top > r.m + kSlack || top_v > r.mv + kSlack))
    {
        const float m = fmaxf(r.m, groups_max(top)), mv = fmaxf(r.mv, groups_max(top_v));
        const float back = mv == r.mv ? 1.f : __builtin_amdgcn_exp2f(r.mv - mv);
        r.l *= m == r.m ? 1.f : __builtin_amdgcn_exp2f(r.m - m);
        r.m = m;
        r.mv = mv;
#pragma unroll
        for (int i = 0; i < N; ++i)
            o[i] *= back;
    }
    // weights are exp2(score - m + lift).  Where that would be below 2^-60 they are 0 in fp16 either way, and only l has to see them
    const float m = r.m == -INFINITY ? 0.f : r.m, lift = fmaxf(lv - ((r.mv == -INFINITY ? 0.f : r.mv) - m), -60.f) + kPShift, shift = lift - m;
    float sum = 0.f;
    u32x4 p[2];
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], f, shift)), b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], f, shift));
        sum += a + b;
        p[i >> 2][i & 3] = pack_f16(a, b);
    }
    r.l += sum * __builtin_amdgcn_exp2f(-lift);
    w[0] = join(p[0]);
    w[1] = join(p[1]);
}

template <int DIM, int NW>
struct RowsLds
{
    static constexpr int kLine = DIM + 4;
    static constexpr int kBytes = (NW / 2 * 16 * kLine + NW * 48) * 4;
};

// 16 rows (`tile`) of a request and key head, keys of one part
template <int DIM, bool BF16, bool FP8, int NW>
__device__ __forceinline__ void rows_body(const tllm_paged_attention_params_t& p, const int shift, const Split& split, const Request& req, int head, int b, int tile, int part,
    float* lds)
{
    constexpr int kSteps = DIM / 32, kOut = DIM / 16, kLine = RowsLds<DIM, NW>::kLine, kPlaces = NW / 2;
    float(*acc)[16][kLine] = reinterpret_cast<float(*)[16][kLine]>(lds);
    float(*ms)[16] = reinterpret_cast<float(*)[16]>(lds + kPlaces * 16 * kLine);
    float(*ls)[16] = ms + NW;
    float(*mvs)[16] = ls + NW;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int group = p.q_heads / p.kv_heads;
    const int rows = min(req.rows, p.max_new) * group, row = tile * 16 + r;
    const int first = req.len - req.rows; // position of the request's first row
    const bool live = row < rows;
    const int token = row / group, qh = head * group + row - token * group;
    const int seen = live ? first + token + 1 : 0x7fffffff; // keys [from, seen) are visible to the lane's row; a row that is none masks nothing
    const int from = live && p.window > 0 ? seen - p.window : 0;
    const int last = min(tile * 16 + 15, rows - 1) / group;
    const int lo = p.window > 0 ? max(0, first + tile * 16 / group + 1 - p.window) : 0, hi = first + last + 1;
    const int t_lo = lo / kTile, n_tiles = max(0, (hi + kTile - 1) / kTile - t_lo), per = (n_tiles + split.parts - 1) / split.parts;
    const int t_begin = t_lo + min(n_tiles, part * per), t_end = t_lo + min(n_tiles, (part + 1) * per);

    const int page = 1 << shift;
    const uint32_t head_bytes = page * DIM, side_bytes = head_bytes * p.kv_heads; // at most 32 MB
    const uint8_t* const pool = static_cast<const uint8_t*>(p.pool) + (int64_t) head * head_bytes;
    const int32_t* const table = p.block_table + (int64_t) b * p.table_stride;

    // What a tile needs of memory, each part sent for as soon as its registers are free: blocks two tiles ahead, keys and scales behind the
    // first product, values behind the second.
    int kb = -1, vb = -1; // blocks of the lane's 16 keys in the first and the second product, -1: none
    u32x4 kw[4][DIM / 64], vw[kOut];
    float ks_next = 0.f, vs_next = 0.f;
    auto blocks_of = [&](int t) {
        const int kk = t * kTile + 16 * (r >> 2), vk = t * kTile + 16 * g;
        kb = kk < req.len ? table[kk >> shift] : -1;
        vb = vk < req.len ? table[vk >> shift] : -1;
    };
    auto held = [&](int block) { return (uint32_t) block < (uint32_t) p.num_blocks; };
    auto fetch_keys = [&](int t) {
        const uint8_t* const at = pool + (uint64_t) (uint32_t) (held(kb) ? kb : 0) * (2 * side_bytes) + (((t * kTile + 16 * (r >> 2)) & (page - 1)) + (r & 3)) * DIM + 16 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < DIM / 64; ++j)
                kw[i][j] = *reinterpret_cast<const u32x4*>(at + 4 * i * DIM + 64 * j);
        const float* const s_at = p.scales + (uint64_t) (uint32_t) (held(vb) ? vb : 0) * (uint32_t) (2 * p.kv_heads) + head;
        ks_next = s_at[0];
        vs_next = s_at[p.kv_heads];
    };
    auto fetch_values = [&](int t, int block) {
        const uint8_t* const at = pool + (uint64_t) (uint32_t) (held(block) ? block : 0) * (2 * side_bytes) + side_bytes + r * page + ((t * kTile + 16 * g) & (page - 1));
#pragma unroll
        for (int i = 0; i < kOut; ++i)
            vw[i] = *reinterpret_cast<const u32x4*>(at + 16 * i * page);
    };
    const int t0 = t_begin + wave;
    int vb_now = -1;
    if (t0 < t_end)
    {
        blocks_of(t0);
        vb_now = vb;
        fetch_keys(t0);
        fetch_values(t0, vb_now);
        if (t0 + NW < t_end)
            blocks_of(t0 + NW);
    }
    f16x8 q[kSteps];
    const uint16_t* const q_row = live ? static_cast<const uint16_t*>(p.q) + (req.row0 + token) * p.q_row + qh * p.q_head : nullptr;
    const float factor = load_query<DIM, BF16>(q, q_row, g) * p.scale * kLog2e;

    f32x4 o[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i)
        o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    Seen row_seen;
    // The last tile of a wave sends for nothing.  It is a body of its own: with the loads under a condition inside one loop hipcc 7.2 takes registers of the
    // values that are still to be read for the exponentials (heads of 64, behind `cut`); a test looks for that in the assembly.
    auto step = [&](int t, auto more) {
        const int vk = t * kTile + 16 * g;
        const bool v_in = held(vb_now);
        const float ks = v_in ? ks_next : 0.f, vs = v_in ? vs_next : 0.f;
        float s[16];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < DIM / 64; ++j)
            {
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(kw[i][j][0], kw[i][j][1]), q[2 * j], c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(kw[i][j][2], kw[i][j][3]), q[2 * j + 1], c, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[4 * i + e] = c[e];
        }
        const int vb_next = vb;
        if constexpr (more)
        {
            fetch_keys(t + NW);
            if (t + 2 * NW < t_end)
                blocks_of(t + 2 * NW);
        }
        const int keep = v_in ? req.len - vk : 0;
        f16x8 w[2];
        soften(s, w, row_seen, o, ks, __builtin_amdgcn_logf(vs), factor, __builtin_amdgcn_ballot_w64(!v_in || vk + 16 > seen || vk < from) == 0, v_in, vk, from, seen);
        if (__builtin_amdgcn_ballot_w64(keep < 16))
#pragma unroll
            for (int i = 0; i < kOut; ++i)
                vw[i] = cut(vw[i], keep);
#pragma unroll
        for (int i = 0; i < kOut; ++i)
        {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(vw[i][0], vw[i][1]), w[0], o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight<FP8>(vw[i][2], vw[i][3]), w[1], o[i], 0, 0, 0);
        }
        vb_now = vb_next;
        if constexpr (more)
            fetch_values(t + NW, vb_now);
    };
    if (t0 < t_end)
    {
        int t = t0;
        for (; t + NW < t_end; t += NW)
            step(t, std::true_type{});
        step(t, std::false_type{});
    }

    // the waves' parts -> one
    const float l = groups_sum(row_seen.l);
    if (g == 0)
    {
        ms[wave][r] = row_seen.m;
        ls[wave][r] = l;
        mvs[wave][r] = row_seen.mv;
    }
    __syncthreads();
    float mv_all = mvs[0][r];
#pragma unroll
    for (int w = 1; w < NW; ++w)
        mv_all = fmaxf(mv_all, mvs[w][r]);
    const float mine = part_of(row_seen.mv, mv_all);
    if (wave >= kPlaces)
#pragma unroll
        for (int i = 0; i < kOut; ++i)
            *reinterpret_cast<f32x4*>(&acc[wave - kPlaces][r][16 * i + 4 * g]) = o[i] * mine;
    __syncthreads();
    if (wave < kPlaces)
#pragma unroll
        for (int i = 0; i < kOut; ++i)
        {
            f32x4* const at = reinterpret_cast<f32x4*>(&acc[wave][r][16 * i + 4 * g]);
            *at = *at + o[i] * mine;
        }
    __syncthreads();
    for (int u = tid; u < 16 * DIM / 4; u += 64 * NW)
    {
        const int ur = u / (DIM / 4), d = u % (DIM / 4) * 4, urow = tile * 16 + ur;
        if (urow >= rows)
            continue;
        float um = ms[0][ur], umv = mvs[0][ur];
#pragma unroll
        for (int w = 1; w < NW; ++w)
        {
            um = fmaxf(um, ms[w][ur]);
            umv = fmaxf(umv, mvs[w][ur]);
        }
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w)
            sum += ls[w][ur] * __builtin_amdgcn_exp2f(ms[w][ur] - (um == -INFINITY ? 0.f : um));
        f32x4 a = *reinterpret_cast<const f32x4*>(&acc[0][ur][d]);
#pragma unroll
        for (int i = 1; i < kPlaces; ++i)
            a += *reinterpret_cast<const f32x4*>(&acc[i][ur][d]);
        const int utoken = urow / group, uh = head * group + urow - utoken * group;
        if (split.parts > 1)
        {
            const int64_t at = split.at(b, req.row0, utoken, p.q_heads, uh) + part;
            *reinterpret_cast<f32x4*>(split.o + at * DIM + d) = a;
            if (d == 0)
                split.seen[at] = make_float4(um, sum, umv, 0.f);
            continue;
        }
        const float to = result_of(um, umv, sum);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (req.row0 + utoken) * p.out_row + uh * p.out_head + d)
            = make_uint2(pack_out<BF16>(a[0] * to, a[1] * to), pack_out<BF16>(a[2] * to, a[3] * to));
    }
}

// a workgroup per request, key head and part of the keys: rows of one tile
template <int DIM, bool BF16, bool FP8, int NW>
__global__ __launch_bounds__(64 * NW) void rows_kernel(const tllm_paged_attention_params_t p, const int shift, const Split split)
{
    __shared__ f32x4 lds[RowsLds<DIM, NW>::kBytes / 16];
    int id = blockIdx.x;
    const int part = id % split.parts;
    id /= split.parts;
    const int head = id % p.kv_heads, b = id / p.kv_heads;
    const Request req = request_of(p, b, shift);
    if (req.rows > 0)
        rows_body<DIM, BF16, FP8, NW>(p, shift, split, req, head, b, 0, part, reinterpret_cast<float*>(lds));
}

template <int DIM>
struct TileForm
{
    static constexpr int kRt = DIM == 256 ? 1 : 2, kRows = 64 * kRt; // row tiles of a wave, rows of a workgroup of four
    static constexpr int kKeyFrags = 4 * DIM / 32, kFrags = 2 * kKeyFrags; // of 1 KB: keys [part][k-step], values [channels / 16][k-step]
    static constexpr int kAhead = DIM == 256 ? 2 : 4; // fragments that are read ahead of their products
    // Tiles that LDS holds: two, one computed and one arriving; of heads of 256 one, so that two workgroups fit a CU (with 30 to 60 registers a lane
    // spilled; 1024 tokens behind 1500, 32 heads: 98 us, one workgroup a half more)
    static constexpr int kBuffers = DIM == 256 ? 1 : 2, kLds = kBuffers * kFrags * 1024;
};

// Tiles of kRows rows of a request and key head.  Requests of at most 16 rows in the same batch take rows_body, in the first light_groups workgroups,
// or in those of their tile 0 if there are none.
template <int DIM, bool BF16, bool FP8>
__global__ __launch_bounds__(256, DIM == 64 ? 3 : 2) void tile_kernel(const tllm_paged_attention_params_t p, const int shift, const int row_tiles, const int light_groups, const Split light,
    const Split split)
{
    using F = TileForm<DIM>;
    constexpr int kSteps = DIM / 32, kOut = DIM / 16, RT = F::kRt;
    extern __shared__ u32x4 frags[]; // [kBuffers][kFrags][64]
    // Workgroups go round the XCDs.  Those of an XCD take the row tiles of as many pairs of request and key head as fill its places, then the next
    // ones': the tiles of a pair walk its keys side by side, which the XCD's L2 holds, and the tiles with the most keys begin first, so that
    // the last ones to begin are short (12 requests of up to 700, 32 heads of 128: 117 us, 125 pair after pair; 4 of 1024 behind 3000, 32 heads on 8: 223, 234).  Where
    // every tile has a place from the start, the second half comes the other way round: workgroups 32 apart of an XCD meet on one CU, a light one
    // beside a heavy one (2048 tokens behind 1500, 32 heads of 128: 114 us, 116 without, 126 pair after pair; heads of 64: 79, 82, 91).
    const int group_id = blockIdx.z * gridDim.x + blockIdx.x; // a launch of many workgroups goes on in z
    const int id = group_id - light_groups, xcd = id & 7, pairs8 = (p.n_seqs * p.kv_heads + 7) >> 3, mine = pairs8 * row_tiles;
    if (id >= 8 * mine)
        return;
    const int at8 = mine <= 64 && id >> 3 >= 32 ? 32 + mine - 1 - (id >> 3) : id >> 3;
    const int most = max(1, 64 / row_tiles), turn = at8 / (most * row_tiles), in = at8 - turn * (most * row_tiles), width = min(most, pairs8 - turn * most);
    const int tile = id < 0 ? 0 : row_tiles - 1 - in / width;
    const int part = id < 0 ? group_id % light.parts : blockIdx.y, pair = id < 0 ? group_id / light.parts : (turn * most + in % width) * 8 + xcd;
    if (pair >= p.n_seqs * p.kv_heads)
        return;
    const int head = pair % p.kv_heads, b = pair / p.kv_heads, group = p.q_heads / p.kv_heads;
    const Request req = request_of(p, b, shift);
    const int rows = min(req.rows, p.max_new) * group;
    if (tile * F::kRows >= rows)
        return;
    if (rows <= 16)
    {
        if (blockIdx.y == 0 && (id < 0 || light_groups == 0))
            rows_body<DIM, BF16, FP8, 4>(p, shift, light, req, head, b, 0, part, reinterpret_cast<float*>(frags));
        return;
    }
    if (id < 0)
        return;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int first = req.len - req.rows;
    // tiles of keys that rows [a, a + n) see
    auto tiles_lo = [&](int a) { return p.window > 0 ? max(0, first + a / group + 1 - p.window) / kTile : 0; };
    auto tiles_hi = [&](int a, int n) { return (max(0, first + min(a + n - 1, rows - 1) / group + 1) + kTile - 1) / kTile; };
    const int row0 = tile * F::kRows, t_lo = tiles_lo(row0), n_tiles = max(0, tiles_hi(row0, F::kRows) - t_lo), per = (n_tiles + split.parts - 1) / split.parts;
    const int t_begin = t_lo + min(n_tiles, part * per), t_end = t_lo + min(n_tiles, (part + 1) * per);
    const int my0 = row0 + wave * 16 * RT;
    const bool idle = my0 >= rows;
    const int my_begin = idle ? t_end : tiles_lo(my0), my_end = idle ? t_end : tiles_hi(my0, 16 * RT);

    const int page = 1 << shift;
    const uint32_t head_bytes = page * DIM, side_bytes = head_bytes * p.kv_heads; // at most 32 MB
    const uint8_t* const pool = static_cast<const uint8_t*>(p.pool) + (int64_t) head * head_bytes;
    const int32_t* const table = p.block_table + (int64_t) b * p.table_stride;
    auto held = [&](int block) { return (uint32_t) block < (uint32_t) p.num_blocks; };

    // The wave brings part `wave` of the keys and channels 16 (wave + 4 i) of the values, 16 bytes a lane and load, as rows_body reads them.
    int kb = -1, vb = -1;
    u32x4 kw[DIM / 64], vw[DIM / 64];
    float ks_next = 0.f, vs_next = 0.f;
    int vb_there = -1; // blocks of what has been sent for
    auto blocks_of = [&](int t) {
        const int kk = t * kTile + 16 * (r >> 2), vk = t * kTile + 16 * g;
        kb = kk < req.len ? table[kk >> shift] : -1;
        vb = vk < req.len ? table[vk >> shift] : -1;
    };
    auto send = [&](int t) {
        const uint8_t* const ka = pool + (uint64_t) (uint32_t) (held(kb) ? kb : 0) * (2 * side_bytes) + (((t * kTile + 16 * (r >> 2)) & (page - 1)) + (r & 3) + 4 * wave) * DIM + 16 * g;
        const uint8_t* const va = pool + (uint64_t) (uint32_t) (held(vb) ? vb : 0) * (2 * side_bytes) + side_bytes + (16 * wave + r) * page + ((t * kTile + 16 * g) & (page - 1));
#pragma unroll
        for (int j = 0; j < DIM / 64; ++j)
        {
            kw[j] = *reinterpret_cast<const u32x4*>(ka + 64 * j);
            vw[j] = *reinterpret_cast<const u32x4*>(va + 64 * j * page);
        }
        const float* const s_at = p.scales + (uint64_t) (uint32_t) (held(vb) ? vb : 0) * (uint32_t) (2 * p.kv_heads) + head;
        ks_next = s_at[0];
        vs_next = s_at[p.kv_heads];
        vb_there = vb;
    };
    auto land = [&](int t) {
        u32x4* const to = frags + (t & (F::kBuffers - 1)) * F::kFrags * 64 + lane;
        const int keep = held(vb_there) ? req.len - (t * kTile + 16 * g) : 0;
        const bool whole = __builtin_amdgcn_ballot_w64(keep < 16) == 0;
#pragma unroll
        for (int j = 0; j < DIM / 64; ++j)
        {
            u32x4* const kt = to + (wave * kSteps + 2 * j) * 64;
            kt[0] = __builtin_bit_cast(u32x4, eight<FP8>(kw[j][0], kw[j][1]));
            kt[64] = __builtin_bit_cast(u32x4, eight<FP8>(kw[j][2], kw[j][3]));
            u32x4 v = vw[j];
            if (!whole)
                v = cut(v, keep);
            u32x4* const vt = to + (F::kKeyFrags + (wave + 4 * j) * 2) * 64;
            vt[0] = __builtin_bit_cast(u32x4, eight<FP8>(v[0], v[1]));
            vt[64] = __builtin_bit_cast(u32x4, eight<FP8>(v[2], v[3]));
        }
    };

    f16x8 q[RT][kSteps];
    f32x4 o[RT][kOut];
    float factor[RT];
    Seen rows_seen[RT];
    int seen[RT], from[RT];
    if (t_begin < t_end)
    {
        blocks_of(t_begin);
        send(t_begin);
        if (t_begin + 1 < t_end)
            blocks_of(t_begin + 1);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        const int row = my0 + 16 * i + r, token = row / group, qh = head * group + row - token * group;
        const bool live = row < rows;
        const uint16_t* const q_row = live ? static_cast<const uint16_t*>(p.q) + (req.row0 + token) * p.q_row + qh * p.q_head : nullptr;
        factor[i] = load_query<DIM, BF16>(q[i], q_row, g) * p.scale * kLog2e;
        seen[i] = live ? first + token + 1 : 0x7fffffff;
        from[i] = live && p.window > 0 ? seen[i] - p.window : 0;
#pragma unroll
        for (int d = 0; d < kOut; ++d)
            o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float ks = 0.f, vs = 0.f;
    bool v_in = false;
    if (t_begin < t_end)
    {
        land(t_begin);
        v_in = held(vb_there);
        ks = v_in ? ks_next : 0.f;
        vs = v_in ? vs_next : 0.f;
    }
    __syncthreads();
    auto step = [&](int t, auto more) { // the last one by itself, as in rows_body
        if constexpr (more)
        {
            send(t + 1);
            if (t + 2 < t_end)
                blocks_of(t + 2);
        }
        if (t >= my_begin && t < my_end)
        {
            const u32x4* const kt = frags + (t & (F::kBuffers - 1)) * F::kFrags * 64 + lane;
            const u32x4* const vt = kt + F::kKeyFrags * 64;
            const int vk = t * kTile + 16 * g;
            f32x4 c[RT][4];
            // fragments are read kAhead before their products: LDS answers behind some hundred cycles
            constexpr int kAhead = F::kAhead;
            float s[RT][16];
            u32x4 a[2][kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                a[0][j] = kt[j * 64];
#pragma unroll
            for (int i = 0; i < F::kKeyFrags / kAhead; ++i)
            {
                if (i + 1 < F::kKeyFrags / kAhead)
#pragma unroll
                    for (int j = 0; j < kAhead; ++j)
                        a[(i + 1) & 1][j] = kt[((i + 1) * kAhead + j) * 64];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                {
                    const int part = (kAhead * i + j) / kSteps, step = (kAhead * i + j) % kSteps;
#pragma unroll
                    for (int n = 0; n < RT; ++n)
                        c[n][part] = __builtin_amdgcn_mfma_f32_16x16x32_f16(join(a[i & 1][j]), q[n][step], step ? c[n][part] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int n = 0; n < RT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[n][i] = c[n][i / 4][i % 4];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                a[0][j] = vt[j * 64];
            const float lv = __builtin_amdgcn_logf(vs);
            f16x8 w[RT][2];
#pragma unroll
            for (int n = 0; n < RT; ++n)
                soften(s[n], w[n], rows_seen[n], o[n], ks, lv, factor[n], __builtin_amdgcn_ballot_w64(!v_in || vk + 16 > seen[n] || vk < from[n]) == 0, v_in, vk, from[n], seen[n]);
#pragma unroll
            for (int i = 0; i < F::kKeyFrags / kAhead; ++i) // as many fragments of values: channels 16 (f / 2), keys 32 (f % 2)
            {
                if (i + 1 < F::kKeyFrags / kAhead)
#pragma unroll
                    for (int j = 0; j < kAhead; ++j)
                        a[(i + 1) & 1][j] = vt[((i + 1) * kAhead + j) * 64];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
#pragma unroll
                    for (int n = 0; n < RT; ++n)
                    {
                        f32x4& to = o[n][(kAhead * i + j) / 2];
                        to = __builtin_amdgcn_mfma_f32_16x16x32_f16(join(a[i & 1][j]), w[n][j & 1], to, 0, 0, 0);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (more)
        {
            if constexpr (F::kBuffers == 1)
                __syncthreads(); // every wave has read the tile
            land(t + 1); // two buffers: its one was read in the round before
            v_in = held(vb_there);
            ks = v_in ? ks_next : 0.f;
            vs = v_in ? vs_next : 0.f;
            __syncthreads();
        }
    };
    if (t_begin < t_end)
    {
        for (int t = t_begin; t + 1 < t_end; ++t)
            step(t, std::true_type{});
        step(t_end - 1, std::false_type{});
    }
#pragma unroll
    for (int n = 0; n < RT; ++n)
    {
        const float sum = groups_sum(rows_seen[n].l);
        const int row = my0 + 16 * n + r, token = row / group, qh = head * group + row - token * group;
        if (row >= rows)
            continue;
        if (split.parts > 1)
        {
            const int64_t at = split.at(b, req.row0, token, p.q_heads, qh) + part;
#pragma unroll
            for (int d = 0; d < kOut; ++d)
                *reinterpret_cast<f32x4*>(split.o + at * DIM + 16 * d + 4 * g) = o[n][d];
            if (g == 0)
                split.seen[at] = make_float4(rows_seen[n].m, sum, rows_seen[n].mv, 0.f);
            continue;
        }
        const float by = result_of(rows_seen[n].m, rows_seen[n].mv, sum);
        uint16_t* const to = static_cast<uint16_t*>(p.out) + (req.row0 + token) * p.out_row + qh * p.out_head + 4 * g;
#pragma unroll
        for (int d = 0; d < kOut; ++d)
            *reinterpret_cast<uint2*>(to + 16 * d) = make_uint2(pack_out<BF16>(o[n][d][0] * by, o[n][d][1] * by), pack_out<BF16>(o[n][d][2] * by, o[n][d][3] * by));
    }
}

// Parts of the keys -> rows: a workgroup per row and head, `per` rows a request; its waves take the parts in turn.
template <int DIM, bool BF16>
__global__ __launch_bounds__(256) void merge_kernel(const tllm_paged_attention_params_t p, const int shift, const int per, const Split light, const Split heavy)
{
    constexpr int kPer = DIM / 64;
    __shared__ float os[4][DIM];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = blockIdx.x;
    const int h = id % p.q_heads;
    id /= p.q_heads;
    const int i = id % per, b = id / per;
    float4 seen;           // of part `lane`: there are 64 at most
    float x[4][kPer] = {}; // four parts of a wave at a time
    auto send = [&](const Split& split, int64_t at, int s0) {
        if (s0 == 0) // every lane: what one split has sent for is nothing of the other
            seen = lane < split.parts ? split.seen[at + lane] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const int s = s0 + 4 * k + wave;
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                x[k][e] = s < split.parts ? split.o[(at + s) * DIM + lane * kPer + e] : 0.f;
        }
    };
    // where the parts of a request of one tile lie does not hang on the request: they are sent for before it is known to be one
    const int64_t at_light = light.at(b, 0, i, p.q_heads, h);
    if (light.parts > 1 && i < light.per)
        send(light, at_light, 0);
    const Request req = request_of(p, b, shift);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            asm volatile("" : "+v"(x[k][e])); // and not behind the branch
    const bool few = min(req.rows, p.max_new) * (p.q_heads / p.kv_heads) <= 16;
    const Split split = few ? light : heavy;
    if (i >= req.rows || split.parts == 1)
        return;
    const int64_t at = few ? at_light : heavy.at(b, req.row0, i, p.q_heads, h);
    if (!few)
        send(heavy, at, 0);
    const float m = wave_max(seen.x), mv = wave_max(seen.z), w = part_of(seen.z, mv);
    const float by = result_of(m, mv, wave_sum(seen.y * __builtin_amdgcn_exp2f(seen.x - (m == -INFINITY ? 0.f : m))));
    float o[kPer] = {};
    for (int s0 = 0;;)
    {
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const float ws = __shfl(w, min(s0 + 4 * k + wave, 63), 64);
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                o[e] += ws * x[k][e];
        }
        s0 += 16;
        if (s0 >= split.parts)
            break;
        send(split, at, s0);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e)
        os[wave][lane * kPer + e] = o[e];
    __syncthreads();
    for (int d = threadIdx.x; d < DIM; d += 256)
    {
        const float v = (os[0][d] + os[1][d] + os[2][d] + os[3][d]) * by;
        static_cast<uint16_t*>(p.out)[(req.row0 + i) * p.out_row + h * p.out_head + d] = BF16 ? f2bf(v) : f2h(v);
    }
}

bool one_tile(const tllm_paged_attention_params_t& p) // no request has more than 16 rows of a key head
{
    return (int64_t) p.max_new * (p.q_heads / p.kv_heads) <= 16;
}

int row_tiles_of(const tllm_paged_attention_params_t& p) // of tile_kernel
{
    const int rows = p.head_size == 256 ? TileForm<256>::kRows : TileForm<128>::kRows;
    return (int) (((int64_t) p.max_new * (p.q_heads / p.kv_heads) + rows - 1) / rows);
}

// Workgroups that the keys are split into.
// Requests of one tile of rows: with fewer requests and key heads than CUs two a CU.  With more of them the split only evens out contexts of
// different lengths, and joining costs more than that unless they are long (64 x 8 heads over 300 to 600 keys of 128: 21 us whole, 28 in
// two parts; 48 x 8 over 4000 to 8000: 115 in three, 126 whole; one of 32 heads over 1032: 10.7 in 8 parts, 12.4 in 4).  The host does not know
// how many such requests there are among prompts: at most as many as leave the others no more than max_new rows each (4 tokens over 30000 keys beside a prompt of 1024, 32 heads
// on 8: 76 us, 338 with their keys whole; tokens alone 44, the prompt alone 36).
// More rows: what fills two places on every CU, where their tiles do not (443 tokens of one head over 57000 keys: 7 tiles).
struct Parts
{
    int waves; // of rows_kernel
    int light, heavy, per; // of requests of one tile of rows, of the others; rows that one of the light ones has at most
};
Parts parts_of(const tllm_paged_attention_params_t& p)
{
    const int64_t pairs = (int64_t) p.n_seqs * p.kv_heads, cus = launch_util::device_cus();
    const int64_t keys = p.window > 0 ? std::min<int64_t>((int64_t) p.window + p.max_new, p.max_kv) : p.max_kv;
    auto within = [](int64_t want, int64_t most) { return (int) std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 64)); };
    Parts s = {4, 1, 1, std::min(p.max_new, 16 / (p.q_heads / p.kv_heads))};
    int64_t few = pairs, least = pairs >= cus ? 2048 : pairs * 4 >= cus ? 512 : 128;
    if (!one_tile(p))
    {
        s.heavy = within(2 * cus / (pairs * row_tiles_of(p)), keys / 1024);
        few = s.per ? std::min<int64_t>(p.n_seqs - 1, ((int64_t) p.n_seqs * p.max_new - p.n_rows) / (p.max_new - s.per)) * p.kv_heads : 0;
        least = 1024;
    }
    if (few > 0 && (int64_t) p.n_seqs * s.per * p.q_heads <= 1 << 23) // what merge_kernel's launch takes
        s.light = within(((few < cus ? 2 : 4) * cus + few - 1) / few, keys / least);
    // Few keys are not split: eight waves of one workgroup and no second launch (500 keys, 32 heads of 128: 9.1 us, 10.0 in parts, 1032: 13.2 and 11.0;
    // 1032 keys, 4 x 8 heads of 64: 8.4 and 9.0, 2048: 11.5 and 10.1).  Heads of 256 have no registers for eight.
    if (one_tile(p) && s.light > 1 && keys * p.head_size <= 65536 && p.head_size < 256)
    {
        s.light = 1;
        s.waves = 8;
    }
    return s;
}

struct Places // rows of the workspace
{
    int64_t light, heavy;
};
Places places_of(const tllm_paged_attention_params_t& p, const Parts& s)
{
    return {s.light > 1 ? (int64_t) p.n_seqs * s.per * p.q_heads * s.light : 0, s.heavy > 1 ? (int64_t) p.n_rows * p.q_heads * s.heavy : 0};
}

template <int DIM, bool BF16, bool FP8>
void launch_form(const tllm_paged_attention_params_t& p, void* workspace, hipStream_t stream)
{
    const int shift = __builtin_ctz((unsigned) p.page_size);
    const int64_t pairs = (int64_t) p.n_seqs * p.kv_heads;
    const Parts s = parts_of(p);
    const auto n = places_of(p, s);
    float* const o = static_cast<float*>(workspace);
    float4* const seen = reinterpret_cast<float4*>(o + (n.light + n.heavy) * DIM);
    const Split light = {o, seen, s.light, s.per}, heavy = {o + n.light * DIM, seen + n.light, s.heavy, 0};
    if (one_tile(p))
    {
        if constexpr (DIM < 256)
            if (s.waves == 8)
            {
                rows_kernel<DIM, BF16, FP8, 8><<<(unsigned) (pairs * s.light), 512, 0, stream>>>(p, shift, light);
                return;
            }
        rows_kernel<DIM, BF16, FP8, 4><<<(unsigned) (pairs * s.light), 256, 0, stream>>>(p, shift, light);
    }
    else
    {
        using F = TileForm<DIM>;
        const int row_tiles = row_tiles_of(p), light_groups = s.light > 1 ? (int) ((pairs * s.light + 7) / 8 * 8) : 0;
        launch_util::ensure_dynamic_lds(reinterpret_cast<const void*>(&tile_kernel<DIM, BF16, FP8>), F::kLds);
        const int64_t all = light_groups + (pairs + 7) / 8 * 8 * row_tiles, wide = std::min<int64_t>(all, 1 << 22); // both multiples of 8; 2^32 threads are too many in x
        tile_kernel<DIM, BF16, FP8><<<dim3((unsigned) wide, s.heavy, (unsigned) ((all + wide - 1) / wide)), 256, F::kLds, stream>>>(p, shift, row_tiles, light_groups, light, heavy);
    }
    const int per = s.heavy > 1 ? p.max_new : s.per;
    if (s.light > 1 || s.heavy > 1)
        merge_kernel<DIM, BF16><<<(unsigned) ((int64_t) p.n_seqs * per * p.q_heads), 256, 0, stream>>>(p, shift, per, light, heavy);
}

template <int DIM, bool BF16>
void launch_dim(const tllm_paged_attention_params_t& p, void* workspace, hipStream_t stream)
{
    if (p.cache_type == TLLM_FP8)
        launch_form<DIM, BF16, true>(p, workspace, stream);
    else
        launch_form<DIM, BF16, false>(p, workspace, stream);
}
} // namespace

size_t paged_attention_workspace(const tllm_paged_attention_params_t& p)
{
    const Places n = places_of(p, parts_of(p));
    return (size_t) (n.light + n.heavy) * (p.head_size + 4) * 4;
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
