// hx_w4.hip -- linear and row lookup over 4-bit weights with group scales (no trellis, no Hadamard) on gfx950.
//
//   weight (n, k) = scales[n][k / group] * (q(n, k) - zeros[n][k / group]),  q in 0..15, zeros 8 where there are none
//
// Words: row n is ceil(K / 128) blocks of 16 uint32; word 4 g + j of a block holds the octet of weights
// k = 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7), nibble 0 (the low bits) first.  So (word >> 4 p) & 0x000f000f is the pair
// k = 2p, 2p + 1 of the octet, and the 16 bytes that a lane loads (words 4 g .. 4 g + 3) are its operands of four
// consecutive 32-k matrix instructions (lane group g of each holds 8 consecutive k): no group of 32 k and more spans two
// instructions, whatever its size.
#include "hx_device.hpp"
#include "hx_kernels.hpp"

namespace hx {

namespace {

// First k, within its row, of word w of a row.
HX_INLINE int word_k(int w) { return (w >> 4) * 128 + 32 * (w & 3) + 8 * ((w >> 2) & 3); }

// q - zero of the 8 weights of a word, in k order.
HX_INLINE void word_values(uint32_t w, float zero, float (&v)[8])
{
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        v[2 * p] = (float)((w >> (4 * p)) & 15u) - zero;
        v[2 * p + 1] = (float)((w >> (4 * p + 16)) & 15u) - zero;
    }
}

}  // namespace

// One wave per output column and 8 rows; a lane takes every 64th word, fp32 sums throughout (the products of an octet
// are summed before the group's scale is applied).
__global__ __launch_bounds__(256) void w4_gemm_kernel(const _Float16* x, W4Args a, void* y, int M, bool y_fp32)
{
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, m0 = 8 * blockIdx.y;
    if (n >= a.N) return;
    const int nw = (a.K + 127) / 128 * 16;
    const uint32_t* wr = a.words + (size_t)n * nw;
    float acc[8] = {};
    for (int w = lane; w < nw; w += 64) {
        const int k = word_k(w);
        if (k >= a.K) continue;
        const size_t g = (size_t)n * a.groups + (k >> a.group_log2);
        float v[8];
        word_values(wr[w], a.zeros ? (float)a.zeros[g] : 8.0f, v);
        const float s = (float)a.scales[g];
#pragma unroll
        for (int m = 0; m < 8; ++m)
            if (m0 + m < M) {
                const hx_h8 xv = *reinterpret_cast<const hx_h8*>(x + (size_t)(m0 + m) * a.K + k);
                float d = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) d += (float)xv[i] * v[i];
                acc[m] += s * d;
            }
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
        float v = acc[m];
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
        if (lane == 0 && m0 + m < M) {
            const size_t i = (size_t)(m0 + m) * a.N + n;
            if (y_fp32) static_cast<float*>(y)[i] = v;
            else static_cast<_Float16*>(y)[i] = (_Float16)v;
        }
    }
}

// out[t][k] = scale * weight(tokens[t], k), the product in fp32 and rounded once; zeros for a token outside [0, N).
// One thread per word: 8 consecutive outputs.
template <typename T>
__global__ __launch_bounds__(256) void w4_embed_kernel(W4Args a, const int64_t* tokens, T* out, long n, float scale)
{
    typedef T v8 __attribute__((ext_vector_type(8)));
    const int nw = (a.K + 127) / 128 * 16;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n * nw) return;
    const long t = i / nw;
    const int w = (int)(i % nw), k = word_k(w);
    if (k >= a.K) return;
    const int64_t row = tokens[t];
    v8 o = {};
    if (row >= 0 && row < a.N) {
        const size_t g = (size_t)row * a.groups + (k >> a.group_log2);
        float v[8];
        word_values(a.words[(size_t)row * nw + w], a.zeros ? (float)a.zeros[g] : 8.0f, v);
        const float s = (float)a.scales[g] * scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (T)(s * v[j]);
    }
    *reinterpret_cast<v8*>(out + (size_t)t * a.K + k) = o;
}

hipError_t launch_w4_gemm(const _Float16* x, const W4Args& a, void* y, int M, bool y_fp32, hipStream_t st)
{
    if (M <= 0 || a.N <= 0) return hipSuccess;
    hipLaunchKernelGGL(w4_gemm_kernel, dim3((a.N + 3) / 4, (M + 7) / 8), dim3(256), 0, st, x, a, y, M, y_fp32);
    return hipGetLastError();
}

hipError_t launch_w4_embed(const W4Args& a, const int64_t* tokens, void* out, long n, float scale, bool out_fp32,
                           hipStream_t st)
{
    if (n <= 0) return hipSuccess;
    const long work = n * ((a.K + 127) / 128 * 16);
    const dim3 grid((unsigned)((work + 255) / 256));
    if (out_fp32)
        hipLaunchKernelGGL((w4_embed_kernel<float>), grid, dim3(256), 0, st, a, tokens, static_cast<float*>(out), n, scale);
    else
        hipLaunchKernelGGL((w4_embed_kernel<_Float16>), grid, dim3(256), 0, st, a, tokens, static_cast<_Float16*>(out), n,
                           scale);
    return hipGetLastError();
}

}  // namespace hx
