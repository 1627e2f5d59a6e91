// Products with 4-bit weights and a scale for each group of a row (tllm_group_matmul): y[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] q[n, k].
//
// v_mfma_f32_16x16x32: A = 16 rows of weights, B = 16 rows of x, so a lane's results are four neighbouring outputs of one row of x.  The
// weights lie in memory as the fragments want them: a tile of 16 rows x 128 k is 1 KB, 16 bytes a lane, word j of a lane the 8 elements of k-step j.
// A k-step is 32 consecutive k of every row, so it lies in one group whatever the group's size; the products of a group are summed by
// themselves and enter the result times the scale in fp32: neither weight nor scale is rounded on the way.
// fp16: nibbles to 1024 + u and 1024 + 16 u by a mask, then u - 8 exactly by a packed subtraction or FMA.  bfloat16 has no packed arithmetic:
// 128 + u goes into the product as it is, and 136 times the sum of the group's x - one more product, with ones for weights - comes off; the difference is up
// to 2^5 smaller than the two, so that it keeps 19 of fp32's 24 bits, where the result keeps 8, and a row with values from 2^113 on comes out as NaN.
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
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <bool BF16>
__device__ __forceinline__ u32x4 weights8(uint32_t w)
{
    u32x4 o;
    if constexpr (BF16) // 128 + u
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    }
    else
    {
        const h2_t low = {(_Float16) -1032.f, (_Float16) -1032.f}, high = {(_Float16) -72.f, (_Float16) -72.f};
        const h2_t part = {(_Float16) 0.0625f, (_Float16) 0.0625f};
        const uint32_t m = 0x64006400u, w8 = w >> 8;
        o[0] = h2_as_u32(u32_as_h2((w & 0x000f000fu) | m) + low);
        o[1] = h2_as_u32(__builtin_elementwise_fma(u32_as_h2((w & 0x00f000f0u) | m), part, high));
        o[2] = h2_as_u32(u32_as_h2((w8 & 0x000f000fu) | m) + low);
        o[3] = h2_as_u32(__builtin_elementwise_fma(u32_as_h2((w8 & 0x00f000f0u) | m), part, high));
    }
    return o;
}

template <bool BF16>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF16>
__device__ __forceinline__ float to_f32(uint32_t bits16)
{
    if constexpr (BF16)
        return bf2f((uint16_t) bits16);
    else
        return h2f((uint16_t) bits16);
}

__device__ __forceinline__ u32x4 as_u32x4(const uint4& v)
{
    return u32x4{v.x, v.y, v.z, v.w};
}

// y += s * (acc - what the raw bfloat16 weights count too much)
template <bool BF16>
__device__ __forceinline__ void scaled_add(f32x4& y, const f32x4& acc, const f32x4& sum, uint2 s)
{
    const float f[4] = {to_f32<BF16>(s.x & 0xffffu), to_f32<BF16>(s.x >> 16), to_f32<BF16>(s.y & 0xffffu), to_f32<BF16>(s.y >> 16)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] += f[i] * (BF16 ? acc[i] - 136.f * sum[i] : acc[i]);
}

template <bool BF16>
__device__ __forceinline__ void store4(const tllm_group_matmul_params_t& p, const f32x4& y, int m, int n)
{
    uint16_t* const to = static_cast<uint16_t*>(p.y) + (int64_t) m * p.ldy;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < p.n)
            to[n + i] = BF16 ? f2bf(y[i]) : f2h(y[i]);
}

__device__ const uint4 kZeros[1] = {};

// 64 lanes x 16 bytes to LDS, lane by lane from lds_byte on; what is under way is counted by hand
__device__ __forceinline__ void dma16(const void* from, uint32_t lds_byte)
{
    uint32_t m0_keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0" : "=&s"(m0_keep) : "v"(from), "s"(lds_byte) : "memory");
}

// 4 R rows x 16 NT outputs a workgroup; its waves share the k-tiles out and join through LDS.  What it has to read is the weights, once;
// each CU also reads all of x, which is as much as its weights at 8 rows and 16 outputs and is why x comes by whole 256-byte pieces of the
// rows that there are.  A wave has a ring of kDeep k-tiles in LDS, its own: no barrier, only the count of what is under way; where LDS holds
// one k-tile a wave, 8 waves with one hide more than 4 with two (64 x 12288 x 4096: 16.3 us, 20.6).  Bound by the weights' bytes and, from 16 rows on, by x
// on its way from L2 (1 x 4096 x 4096 4.7 us, of them 2 the launch and the join; 8 x 4096 x 11008 in bfloat16 8.0; 24 x 12288 x 4096 10.6).
template <int R, int NT>
struct FewForm
{
    static constexpr int kSlot = R + NT + 1; // KB: x, weights, scales
    static constexpr int kWaves = kSlot <= 4 ? 16 : 8, kFit = 160 / (kWaves * kSlot), kDeep = kFit < 4 ? kFit : 4;
    static constexpr int kRing = kWaves * kDeep * kSlot * 1024, kMT = (R + 3) / 4;
    static_assert(kDeep >= 1 && kWaves * kMT * NT * 1024 <= 160 * 1024 && (kDeep - 1) * kSlot < 64, "the ring fits LDS and the counter");
    static constexpr int kLds = kRing > kWaves * kMT * NT * 1024 ? kRing : kWaves * kMT * NT * 1024;
};

template <bool BF16, int GROUP, int R, int NT>
__global__ __launch_bounds__((64 * FewForm<R, NT>::kWaves)) void few_rows_kernel(const tllm_group_matmul_params_t p)
{
    using F = FewForm<R, NT>;
    constexpr int kSteps = GROUP / 32, kGroups = 4 / kSteps, MT = F::kMT, kMask = R < 4 ? 4 * R - 1 : 15;
    extern __shared__ uint4 lds[];
    typedef __attribute__((address_space(3))) void lds_t;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int k_tiles = (p.k + 127) / 128, n_tiles = (p.n + 15) / 16, n_all = n_tiles * 16, n0 = blockIdx.x * NT, m0 = blockIdx.y * 4 * R;
    const int groups = (p.k + GROUP - 1) / GROUP;
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const uint32_t lds0 = (uint32_t) (uintptr_t) (lds_t*) lds + wave * F::kDeep * F::kSlot * 1024;

    auto bring = [&](int slot, int t) {
        const uint32_t to = lds0 + slot * F::kSlot * 1024;
#pragma unroll
        for (int i = 0; i < R; ++i)
        {
            // rows of 256 bytes, piece c of 16 bytes at c ^ row: the 16 rows of a fragment read 16 different places
            const int row = 4 * i + g, k = t * 128 + ((r ^ (row & 15)) << 3);
            const void* from = static_cast<const uint16_t*>(p.x) + (int64_t) min(m0 + row, p.rows - 1) * p.ldx + k;
            dma16(k < p.k ? from : static_cast<const void*>(kZeros), to + i * 1024);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) // a tile behind the last one is computed again and not written
            dma16(static_cast<const uint4*>(p.packed) + ((int64_t) min(n0 + i, n_tiles - 1) * k_tiles + t) * 64 + lane, to + (R + i) * 1024);
        const int piece = min(lane, 2 * NT * kGroups - 1), q = piece / (2 * NT), n = n0 * 16 + (piece - q * 2 * NT) * 8;
        dma16(static_cast<const uint16_t*>(p.scales) + (int64_t) min(t * kGroups + q, groups - 1) * n_all + min(n, n_all - 8), to + (R + NT) * 1024);
    };
    f32x4 y[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
            y[i][j] = zero;
#pragma unroll
    for (int d = 0; d < F::kDeep; ++d)
        if (wave + d * F::kWaves < k_tiles)
            bring(d, wave + d * F::kWaves);
    int slot = 0;
    for (int t = wave; t < k_tiles; t += F::kWaves)
    {
        if (t + (F::kDeep - 1) * F::kWaves < k_tiles)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((F::kDeep - 1) * F::kSlot) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint4* const at = lds + (wave * F::kDeep + slot) * F::kSlot * 64;
#pragma unroll
        for (int q = 0; q < kGroups; ++q)
        {
            u32x4 b[kSteps][MT];
            f32x4 sum[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i)
            {
                sum[i] = zero;
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
                {
                    const int row = r & kMask;
                    b[j][i] = as_u32x4(at[(16 * i + row) * 16 + ((4 * (q * kSteps + j) + g) ^ row)]);
                    if (BF16)
                        sum[i] = product<BF16>(ones, b[j][i], sum[i]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
            {
                const uint32_t* const words = reinterpret_cast<const uint32_t*>(at + (R + n) * 64 + lane) + q * kSteps;
                const uint2 s = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(at + (R + NT) * 64) + (q * NT + n) * 16 + 4 * g);
                f32x4 acc[MT];
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
                {
                    const u32x4 a = weights8<BF16>(words[j]);
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        acc[i] = product<BF16>(a, b[j][i], j ? acc[i] : zero);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    scaled_add<BF16>(y[n][i], acc[i], sum[i], s);
            }
        }
        if (t + F::kDeep * F::kWaves < k_tiles)
        {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the slot is read
            bring(slot, t + F::kDeep * F::kWaves);
        }
        slot = slot + 1 == F::kDeep ? 0 : slot + 1;
    }
    __syncthreads(); // every wave is through with its ring: it takes the sums now
    f32x4* const part = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
            part[(wave * NT * MT + i * MT + j) * 64 + lane] = y[i][j];
    __syncthreads();
    for (int u = wave; u < NT * MT; u += F::kWaves)
    {
        f32x4 v = part[u * 64 + lane];
#pragma unroll
        for (int w = 1; w < F::kWaves; ++w)
            v += part[(w * NT * MT + u) * 64 + lane];
        const int n = (n0 + u / MT) * 16 + 4 * g, m = m0 + u % MT * 16 + r;
        if (m < min(p.rows, m0 + 4 * R)) // fewer than 16 rows: the other lanes computed some of them again
            store4<BF16>(p, v, m, n);
    }
}

// Many rows: 128 rows x 64 NT outputs a workgroup of 8 waves, 64 x 16 NT a wave.  x, weights and scales of a k-tile go to LDS by DMA, x and weights as the
// fragments that the waves read back (64 lanes x 16 bytes in a row: no conflicts), three k-tiles in a ring.
// The two waves of a SIMD are half a k-tile apart: while the one multiplies, converts and scales, the other reads its fragments (in step with each
// other all waves wait for LDS, then all convert, then all multiply: 1024 x 11008 x 4096 122 us, 110 so).  Two barriers a k-tile keep them there, one more at
// the start for the later half and one at the end for the earlier.  Between barriers 2 t - 1 and 2 t the earlier half reads k-tile t, which every
// wave has waited for before barrier 2 t - 1; the later half reads it between 2 t and 2 t + 1; whoever sends for k-tile t + 2 has passed barrier 2 t - 1,
// before which both have read t - 1, whose place it takes.
// 0.84 PFLOP/s; with the matrix instructions alone 1.2, what power leaves of them (a library product of 8192^3: 1.3).
constexpr int kStages = 3;

template <int GROUP, int NT>
struct TileForm
{
    static constexpr int kGroups = 128 / GROUP, kOutTiles = 4 * NT; // tiles of 16 outputs
    static constexpr int kX = 32, kW = kOutTiles, kChunks = kX + kW + kGroups, kPerWave = (kChunks + 7) / 8; // of 1 KB, per k-tile
    static constexpr int kStageBytes = kChunks * 1024;
};

template <bool BF16, int GROUP, int NT>
__global__ __launch_bounds__(512, 2) void tile_kernel(const tllm_group_matmul_params_t p, const int m_tiles, const int tiles)
{
    using F = TileForm<GROUP, NT>;
    constexpr int kSteps = GROUP / 32;
    extern __shared__ uint4 lds[]; // [kStages]: x [8 row tiles][4][64], weights [kOutTiles][64], scales [kGroups][64]
    typedef __attribute__((address_space(3))) void lds_t;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    // workgroups go round the XCDs: each XCD takes a contiguous range of the tiles, whose row tiles share their weights in its L2
    const int q8 = tiles >> 3, r8 = tiles & 7, xcd = blockIdx.x & 7;
    const int id = xcd * q8 + min(xcd, r8) + (blockIdx.x >> 3);
    const int tile_n = id / m_tiles, tile_m = id - tile_n * m_tiles;
    const int k_tiles = (p.k + 127) / 128, n_tiles = (p.n + 15) / 16, n_all = n_tiles * 16, groups = (p.k + GROUP - 1) / GROUP;
    const int wn = wave & 3, wm = wave >> 2, n0 = tile_n * F::kOutTiles;
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const uint32_t lds0 = (uint32_t) (uintptr_t) (lds_t*) lds;

    // A wave brings k-step wave % 4 of row tiles wave / 4 + 2 i, and chunks wave, wave + 8, .. of the weights and then the scales (the last one
    // once more where they do not divide).  Each has an address that moves by the same step every k-tile.
    const int k0 = 32 * (wave & 3) + 8 * g;
    const char* x_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x_at[i] = reinterpret_cast<const char*>(static_cast<const uint16_t*>(p.x) + (int64_t) min((tile_m * 8 + 2 * i + wm) * 16 + r, p.rows - 1) * p.ldx + k0);
    auto bring = [&](int t) {
        const uint32_t to = lds0 + (t % kStages) * F::kStageBytes;
        const bool inside = t * 128 + k0 < p.k; // k may end inside the last k-tile: x is 0 there, as the weights are
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            dma16(inside ? x_at[i] : reinterpret_cast<const char*>(kZeros), to + (i * 8 + wave) * 1024);
            x_at[i] += 256;
        }
#pragma unroll
        for (int i = 0; i < F::kPerWave - 4; ++i)
        {
            const int c = min(i * 8 + wave, F::kW + F::kGroups - 1);
            const char* const at = c < F::kW
                ? static_cast<const char*>(p.packed) + ((int64_t) min(n0 + c, n_tiles - 1) * k_tiles + t) * 1024
                : static_cast<const char*>(p.scales) + (int64_t) min(t * F::kGroups + c - F::kW, groups - 1) * n_all * 2;
            dma16(at + (c < F::kW ? lane * 16 : 2 * min(n0 * 16 + lane * 8, n_all - 8)), to + (F::kX + c) * 1024);
        }
    };
    f32x4 y[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            y[i][j] = zero;

    auto arrived = [&](int t) { // k-tile t of what this wave has sent for, where t + 1 may be under way
        if (t + 1 < k_tiles)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(F::kPerWave) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    auto meet = [&] { // every wave; what this one has read of LDS is there
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    bring(0);
    if (k_tiles > 1)
        bring(1);
    arrived(0);
    meet();
    if (wm)
        meet();
    for (int t = 0; t < k_tiles; ++t)
    {
        if (t + 2 < k_tiles)
            bring(t + 2);
        const uint4* const at = lds + (t % kStages) * (F::kStageBytes / 16);
        const uint4* const xs = at + wm * 4 * 4 * 64 + lane;
        const uint4* const ws = at + (F::kX + wn * NT) * 64 + lane;
        const char* const ss = reinterpret_cast<const char*>(at + (F::kX + F::kW) * 64) + (wn * NT * 16 + 4 * g) * 2;
        u32x4 words[NT], b[4][4];
        uint2 scale[F::kGroups][NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
        {
            words[n] = as_u32x4(ws[n * 64]);
#pragma unroll
            for (int q = 0; q < F::kGroups; ++q)
                scale[q][n] = *reinterpret_cast<const uint2*>(ss + q * 1024 + n * 32);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                b[j][i] = as_u32x4(xs[(i * 4 + j) * 64]);
        if (wm)
            arrived(t + 1);
        meet();
        // Output tile n of group q is u = q NT + n: its products are under way while u + 1 is converted and u - 1 is scaled
        constexpr int kUnits = F::kGroups * NT;
        u32x4 w[2][kSteps];
        f32x4 acc[2][4], sum[2][4];
        auto convert = [&](int u) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
                w[u & 1][j] = weights8<BF16>(words[u % NT][u / NT * kSteps + j]);
        };
        auto add = [&](int u) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                f32x4& to = y[u % NT][i];
                scaled_add<BF16>(to, acc[u & 1][i], sum[u / NT & 1][i], scale[u / NT][u % NT]);
                asm volatile("" : "+v"(to)); // here and not behind the barrier, where every group's products would have to be kept
            }
        };
        convert(0);
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
        {
            const int q = u / NT;
            if (BF16 && u % NT == 0)
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sum[q & 1][i] = product<BF16>(ones, b[q * kSteps + j][i], j ? sum[q & 1][i] : zero);
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[u & 1][i] = product<BF16>(w[u & 1][j], b[q * kSteps + j][i], j ? acc[u & 1][i] : zero);
            if (u > 0)
                add(u - 1);
            if (u + 1 < kUnits)
                convert(u + 1);
        }
        add(kUnits - 1);
        if (!wm)
            arrived(t + 1);
        meet();
    }
    if (!wm)
        meet();
    const bool whole = p.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % 8 == 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const int m = (tile_m * 8 + wm * 4 + i) * 16 + r;
        if (m >= p.rows)
            continue;
#pragma unroll
        for (int j = 0; j < NT; ++j)
        {
            const int n = (n0 + wn * NT + j) * 16 + 4 * g;
            const f32x4 v = y[j][i];
            if (whole && n + 4 <= p.n)
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + (int64_t) m * p.ldy + n)
                    = BF16 ? make_uint2((uint32_t) f2bf(v[0]) | (uint32_t) f2bf(v[1]) << 16, (uint32_t) f2bf(v[2]) | (uint32_t) f2bf(v[3]) << 16)
                           : make_uint2((uint32_t) f2h(v[0]) | (uint32_t) f2h(v[1]) << 16, (uint32_t) f2h(v[2]) | (uint32_t) f2h(v[3]) << 16);
            else if (n < p.n)
                store4<BF16>(p, v, m, n);
        }
    }
}

template <bool BF16, int GROUP, int NT>
void launch_tiles(const tllm_group_matmul_params_t& p, hipStream_t stream)
{
    const size_t lds = kStages * TileForm<GROUP, NT>::kStageBytes;
    const int m_tiles = (p.rows + 127) / 128, n_parts = (p.n + 64 * NT - 1) / (64 * NT);
    launch_util::ensure_dynamic_lds(reinterpret_cast<const void*>(&tile_kernel<BF16, GROUP, NT>), lds);
    tile_kernel<BF16, GROUP, NT><<<m_tiles * n_parts, 512, lds, stream>>>(p, m_tiles, m_tiles * n_parts);
}

template <bool BF16, int GROUP, int R, int NT>
void launch_few(const tllm_group_matmul_params_t& p, hipStream_t stream)
{
    using F = FewForm<R, NT>;
    launch_util::ensure_dynamic_lds(reinterpret_cast<const void*>(&few_rows_kernel<BF16, GROUP, R, NT>), F::kLds);
    const dim3 grid(((p.n + 15) / 16 + NT - 1) / NT, (p.rows + 4 * R - 1) / (4 * R));
    few_rows_kernel<BF16, GROUP, R, NT><<<grid, 64 * F::kWaves, F::kLds, stream>>>(p);
}

// The forms and what a workgroup takes in each (us, all CUs busy): `once` and `each` k-tile, fitted to 256 and 1024 workgroups of fp16 with groups
// of 128 over k of 512 to 11008, which they meet within 10 %; a launch, 1 to 2 us, comes on top (64 x 12288 x 4096: 11.9 by the table, 14.1 measured).  Other types
// and groups choose by the same table, which was not fitted to them: 1024 x 11008 x 4096 takes 112 us, bfloat16 117, with groups of 64 142, of 32 191, and in the
// form 64 x 48, where small groups have no registers left, 128 x 11008 x 4096 takes 26, bfloat16 26, with groups of 64 45, of 32 166.  A product takes as many rounds as its workgroups take CUs, and the form with the
// least time is the one to take: 1 x 4096 x 4096 in 256 workgroups of 16 outputs, 1024 x 11008 x 4096 in 464 tiles of 128 x 192 (109 us; 126 in tiles of
// 128, 136 in tiles of 256, 197 in tiles of 64), 1024 x 4096 x 4096 in 256 of 128 x 128 (44 us; 54 in tiles of 192), 67 x 190 x 10144 in 204 of 4 x 16 (6.5 us; 143 in
// tiles of 192).
struct Form
{
    int rows, outputs;
    float once, each;
};
constexpr Form kForms[] = {{4, 16, 1.0f, .050f}, {4, 32, 1.3f, .077f}, {4, 48, 1.0f, .123f}, {4, 64, 1.1f, .155f}, {8, 16, 1.0f, .057f}, {8, 32, .9f, .097f}, {8, 48, 1.0f, .126f},
    {8, 64, 1.3f, .151f}, {16, 16, .8f, .082f}, {16, 32, 1.1f, .106f}, {16, 48, 1.3f, .131f}, {16, 64, 1.6f, .165f}, {32, 16, 1.1f, .121f}, {32, 32, 1.6f, .151f},
    {32, 48, 2.1f, .183f}, {32, 64, 2.4f, .225f}, {64, 16, 1.9f, .207f}, {64, 32, 2.5f, .229f}, {64, 48, 3.4f, .267f}, {128, 64, 2.5f, .940f}, {128, 128, 4.6f, 1.268f},
    {128, 192, 7.2f, 1.625f}, {128, 256, 8.4f, 2.070f}};

int form_of(int rows, int n, int k)
{
    const int cus = launch_util::device_cus(), k_tiles = (k + 127) / 128;
    int best = 0;
    double least = 1e30;
    for (int i = 0; i < (int) (sizeof(kForms) / sizeof(kForms[0])); ++i)
    {
        const Form& f = kForms[i];
        const int64_t groups = (int64_t) ((n + f.outputs - 1) / f.outputs) * ((rows + f.rows - 1) / f.rows);
        const double us = (double) ((groups + cus - 1) / cus) * ((double) f.once + k_tiles * (double) f.each);
        if (us < least)
        {
            least = us;
            best = i;
        }
    }
    return best;
}

template <bool BF16, int GROUP>
void launch_form(const tllm_group_matmul_params_t& p, hipStream_t stream)
{
    const Form f = kForms[form_of(p.rows, p.n, p.k)];
#define TLLM_FEW(R)                                                                                                    \
    case 4 * R:                                                                                                        \
        f.outputs == 16 ? launch_few<BF16, GROUP, R, 1>(p, stream)                                                     \
            : f.outputs == 32 ? launch_few<BF16, GROUP, R, 2>(p, stream)                                               \
            : f.outputs == 48 ? launch_few<BF16, GROUP, R, 3>(p, stream)                                               \
                              : launch_few<BF16, GROUP, R, (R < 16 ? 4 : 3)>(p, stream);                               \
        break;
    switch (f.rows)
    {
        TLLM_FEW(1)
        TLLM_FEW(2)
        TLLM_FEW(4)
        TLLM_FEW(8)
        TLLM_FEW(16)
    default:
        f.outputs == 64 ? launch_tiles<BF16, GROUP, 1>(p, stream)
            : f.outputs == 128 ? launch_tiles<BF16, GROUP, 2>(p, stream)
            : f.outputs == 192 ? launch_tiles<BF16, GROUP, 3>(p, stream)
                               : launch_tiles<BF16, GROUP, 4>(p, stream);
    }
#undef TLLM_FEW
}
} // namespace

int launch_group_matmul(const tllm_group_matmul_params_t& p, hipStream_t stream)
{
    const bool bf16 = p.dtype == TLLM_BF16;
    switch (p.group)
    {
    case 32: bf16 ? launch_form<true, 32>(p, stream) : launch_form<false, 32>(p, stream); break;
    case 64: bf16 ? launch_form<true, 64>(p, stream) : launch_form<false, 64>(p, stream); break;
    default: bf16 ? launch_form<true, 128>(p, stream) : launch_form<false, 128>(p, stream); break;
    }
    return launched("tllm_group_matmul");
}

} // namespace kernels
} // namespace tllm
