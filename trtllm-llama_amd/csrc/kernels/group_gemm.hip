// Products with 4-bit weights and a scale for each group of a row (tllm_group_matmul): y[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] q[n, k].
//
// v_mfma_f32_16x16x32: A = 16 rows of weights, B = 16 rows of x, so a lane's results are four neighbouring outputs of one row of x.  The
// weights lie in memory as the fragments want them: a tile of 16 rows x 128 k is 1 KB, 16 bytes a lane, word j of a lane the 8 elements of k-step j.
// A k-step is 32 consecutive k of every row, so it lies in one group whatever the group's size; the products of a group are summed by
// themselves and enter the result times the scale in fp32: neither weight nor scale is rounded on the way.
// fp16: nibbles to 1024 + u and 1024 + 16 u by a mask, then u - 8 exactly by a packed subtraction or FMA.  bfloat16 has no packed arithmetic:
// 128 + u goes into the product as it is, and 136 times the sum of the group's x - one more product, with ones for weights - comes off.
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

// 16 outputs x 16 rows a workgroup, its waves take the k-tiles in turn
template <bool BF16, int GROUP>
__global__ __launch_bounds__(256) void rows16_kernel(const tllm_group_matmul_params_t p)
{
    __shared__ f32x4 part[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n_tile = blockIdx.x, m = blockIdx.y * 16 + r, k_tiles = (p.k + 127) / 128, n_all = (p.n + 15) / 16 * 16;
    const uint4* const packed = static_cast<const uint4*>(p.packed) + (int64_t) n_tile * k_tiles * 64 + lane;
    const uint16_t* const scales = static_cast<const uint16_t*>(p.scales) + n_tile * 16 + 4 * g;
    const uint16_t* const x = static_cast<const uint16_t*>(p.x) + (int64_t) min(m, p.rows - 1) * p.ldx + 8 * g;
    constexpr int kSteps = GROUP / 32;
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    for (int t = wave; t < k_tiles; t += 4)
    {
        const uint4 w4 = packed[t * 64];
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        f32x4 acc, sum;
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const int k = t * 128 + j * 32;
            if (k >= p.k)
                break;
            const uint4 x4 = *reinterpret_cast<const uint4*>(x + k);
            const u32x4 b = {x4.x, x4.y, x4.z, x4.w};
            if (j % kSteps == 0)
                acc = sum = f32x4{0.f, 0.f, 0.f, 0.f};
            acc = product<BF16>(weights8<BF16>(w[j]), b, acc);
            if (BF16)
                sum = product<BF16>(ones, b, sum);
            if (j % kSteps == kSteps - 1 || k + 32 >= p.k)
            {
                const uint2 s = *reinterpret_cast<const uint2*>(scales + (int64_t) (k / GROUP) * n_all);
                if (BF16)
                    acc -= 136.f * sum;
                y[0] += to_f32<BF16>(s.x & 0xffffu) * acc[0];
                y[1] += to_f32<BF16>(s.x >> 16) * acc[1];
                y[2] += to_f32<BF16>(s.y & 0xffffu) * acc[2];
                y[3] += to_f32<BF16>(s.y >> 16) * acc[3];
            }
        }
    }
    part[wave][lane] = y;
    __syncthreads();
    if (wave != 0 || m >= p.rows)
        return;
    y = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
    uint16_t* const to = static_cast<uint16_t*>(p.y) + (int64_t) m * p.ldy;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const int n = n_tile * 16 + 4 * g + i;
        if (n < p.n)
            to[n] = BF16 ? f2bf(y[i]) : f2h(y[i]);
    }
}

template <bool BF16, int GROUP>
void launch_form(const tllm_group_matmul_params_t& p, hipStream_t stream)
{
    rows16_kernel<BF16, GROUP><<<dim3((p.n + 15) / 16, (p.rows + 15) / 16), 256, 0, stream>>>(p);
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
