// Root-mean-square norm of x + residual with an 8-bit output.
//
//   h = x + residual;  y = h * rsqrt(mean(h^2) + eps) * weight
//   e = the least integer with max|y| <= 448 * 2^e over each 128 values
//   q = e4m3(y * 2^-e), scale byte e + 127
//
// Bound by memory: x and the residual are read once, the row stays in
// registers through its sum, and the sum and q are written once. A workgroup
// takes a row; a lane holds runs of 8 consecutive values, so that 16 lanes hold
// a block of 128 and its maximum takes four exchanges within a row of lanes.
// Measured: 16384 x 8192 bf16 with the residual 168 us, 940 MB moved (as many
// as there are) at 5.6 TB/s; 1777 x 5001 floats 14.1 us alone and 13.0 us in a
// row of calls, 44 MB at 3.4 TB/s; 1 x 4096 3.3 us.
#include "head_common.h"

#include <math.h>

namespace tkh {

// The largest over the 16 lanes that hold a block (lane / 16 is the block).
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, true)));  // row_ror:8
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xf, 0xf, true)));  // row_ror:4
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xf, 0xf, true)));  // row_ror:2
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x121, 0xf, 0xf, true)));  // row_ror:1
    return v;
}

// The sum over a wave, in every lane.
__device__ __forceinline__ float sum64(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// The sum over a workgroup, in every lane; `part` is used once.
__device__ __forceinline__ float block_sum(float (&part)[16], float v, int t, int threads) {
    v = sum64(v);
    if ((t & 63) == 0) part[t >> 6] = v;
    __syncthreads();
    float sum = 0.0f;
    for (int i = 0; i < threads >> 6; ++i) sum += part[i];
    return sum;
}

// The least e with amax <= 448 * 2^e (448 = 0.875 * 2^9), 0 for a block of
// zeros, within what a scale byte holds.
__device__ __forceinline__ int scale_exponent(float amax) {
    int x;
    float f = frexpf(amax, &x);
    int e = x - 9 + (f > 0.875f ? 1 : 0);
    e = e < -127 ? -127 : e > 127 ? 127 : e;
    return amax > 0.0f ? e : 0;
}

template <typename T, typename W, int VPT>
__global__ __launch_bounds__(1024) void k_norm(const tkh_norm p) {
    typedef typename Raw<T>::type R;
    typedef typename Raw<W>::type RW;
    __shared__ float part[2][16];
    const int64_t row = blockIdx.x;
    const int k = (int)p.k, t = threadIdx.x, threads = blockDim.x;
    const R* x = (const R*)p.x + row * p.x_stride;
    const R* r = p.residual ? (const R*)p.residual + row * p.residual_stride : nullptr;
    R* out = p.residual_out ? (R*)p.residual_out + row * p.out_stride : nullptr;

    float h[VPT][8];
    // the mean is summed in parts of a power of two over 1 / k: what it holds
    // fits wherever the mean does, and no rounding is added
    const int log_k = 32 - __builtin_clz((unsigned)(k - 1) | 1u);
    const float part_k = ldexpf(1.0f, -log_k);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (t + i * threads) * 8;
        R a[8] = {}, b[8] = {};
        if (c + 8 <= k) {
            load_pack(a, x + c);
            if (r) load_pack(b, r + c);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < k) {
                    a[j] = x[c + j];
                    if (r) b[j] = r[c + j];
                }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[i][j] = Num<T>::get(a[j]);
            if (r) h[i][j] += Num<T>::get(b[j]);
            sum += (h[i][j] * part_k) * h[i][j];
        }
        if (out) {
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = Num<T>::put(h[i][j]);
            if (c + 8 <= k) {
                store_pack(out + c, a);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < k) out[c + j] = a[j];
            }
        }
    }
    const float over_k = ldexpf(1.0f, log_k) / (float)k;
    float mean = block_sum(part[0], sum, t, threads) * over_k, eps = p.eps;
    // Where the mean or its sum with eps is infinite, or the mean may have lost
    // squares to underflow and eps does not hide that, it is taken of h times a
    // power of two, and eps with it: the largest such h is below 2^62, and the
    // smallest, of 2^-149, has a square of 2^-106. An h that is infinite itself
    // leaves the mean infinite.
    if (mean + eps == INFINITY || (mean < 0x1p-95f && eps < 0x1p-64f)) {
        const float scale = mean < 1.0f ? 0x1p96f : 0x1p-66f;
        eps = eps * scale * scale;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[i][j] *= scale;
                sum += (h[i][j] * part_k) * h[i][j];
            }
        mean = block_sum(part[1], sum, t, threads) * over_k;
    }
    const float rstd = 1.0f / sqrtf(mean + eps);

    const RW* w = (const RW*)p.weight;
    uint8_t* q = (uint8_t*)p.q + row * p.q_stride;
    uint8_t* scale = (uint8_t*)p.scale + row * p.scale_stride;
    const int padded = (k + kBlock - 1) / kBlock * kBlock;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (t + i * threads) * 8;
        RW a[8] = {};
        if (c + 8 <= k) {
            load_pack(a, w + c);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < k) a[j] = w[c + j];
        }
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[i][j] = h[i][j] * rstd * Num<W>::get(a[j]);
            if (c + j >= k) h[i][j] = 0.0f;  // 0 * inf in the pad
            const float v = fabsf(h[i][j]);
            if (v < INFINITY) amax = fmaxf(amax, v);
        }
        amax = max16(amax);
        const int e = scale_exponent(amax);
        int lo = 0, hi = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = ldexpf(h[i][j], -e);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[i][0], h[i][1], lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[i][2], h[i][3], lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[i][4], h[i][5], hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[i][6], h[i][7], hi, true);
        if (c < padded) {
            *(int2*)(q + c) = make_int2(lo, hi);
            if ((t & 15) == 0) scale[c / kBlock] = (uint8_t)(e + 127);
        }
    }
}

// Lanes of 8 values; past 256 threads a lane takes more of them, so that rows
// of a usual width need one exchange between four waves.
static int runs_a_lane(int64_t k) {
    const int64_t runs = ceil_div(k, 8);
    return runs <= 256 ? 1 : runs <= 512 ? 2 : runs <= 4096 ? 4 : 8;
}
static unsigned threads_of(int64_t k) {
    return (unsigned)(ceil_div(ceil_div(ceil_div(k, 8), runs_a_lane(k)), 64) * 64);
}

template <typename T, typename W> static int norm_rows(const tkh_norm& p, void* stream) {
    const dim3 grid((unsigned)p.rows), block(threads_of(p.k));
    switch (runs_a_lane(p.k)) {
    case 1: return launch("k_norm", k_norm<T, W, 1>, grid, block, 0, stream, p);
    case 2: return launch("k_norm", k_norm<T, W, 2>, grid, block, 0, stream, p);
    case 4: return launch("k_norm", k_norm<T, W, 4>, grid, block, 0, stream, p);
    default: return launch("k_norm", k_norm<T, W, 8>, grid, block, 0, stream, p);
    }
}

}  // namespace tkh

extern "C" int tk_head_norm(const tkh_norm* args, void* stream) {
    using namespace tkh;
    if (!args) return fail(TKH_E_INVALID_ARG, "no arguments");
    const tkh_norm& p = *args;
    if (p.rows < 0 || p.k < 1) return fail(TKH_E_SHAPE, "rows %lld, k %lld", (long long)p.rows, (long long)p.k);
    if (p.k > TKH_NORM_MAX_K)
        return fail(TKH_E_UNSUPPORTED, "k %lld is over %d", (long long)p.k, TKH_NORM_MAX_K);
    if (!fits_launch(p.rows, threads_of(p.k)))
        return fail(TKH_E_SHAPE, "rows %lld of k %lld", (long long)p.rows, (long long)p.k);
    if (p.dtype < TKH_F32 || p.dtype > TKH_F16) return fail(TKH_E_UNSUPPORTED, "dtype %d", p.dtype);
    if (p.weight_dtype != p.dtype && p.weight_dtype != TKH_F32)
        return fail(TKH_E_UNSUPPORTED, "weight dtype %d with dtype %d", p.weight_dtype, p.dtype);
    if (p.rows == 0) return TKH_OK;
    if (!p.x || !p.weight || !p.q || !p.scale) return fail(TKH_E_INVALID_ARG, "a null pointer");
    const int64_t padded = ceil_div(p.k, kBlock) * kBlock;
    if (p.q_stride % 16 || p.q_stride < padded || (uintptr_t)p.q % 16)
        return fail(TKH_E_SHAPE, "rows of q are 16-byte aligned and at least %lld long", (long long)padded);
    if (p.scale_stride < padded / kBlock)
        return fail(TKH_E_SHAPE, "scale rows of %lld", (long long)p.scale_stride);
    if (p.rows > 1 && (p.x_stride < 0 || (p.residual && p.residual_stride < 0) ||
                       (p.residual_out && p.out_stride < p.k)))
        return fail(TKH_E_SHAPE, "a row stride");
    DeviceScope scope(p.device);
    if (scope.status() != TKH_OK) return scope.status();
    if (p.dtype == TKH_F32) return norm_rows<float, float>(p, stream);
    if (p.dtype == TKH_BF16)
        return p.weight_dtype == TKH_F32 ? norm_rows<__hip_bfloat16, float>(p, stream)
                                         : norm_rows<__hip_bfloat16, __hip_bfloat16>(p, stream);
    return p.weight_dtype == TKH_F32 ? norm_rows<__half, float>(p, stream)
                                     : norm_rows<__half, __half>(p, stream);
}
