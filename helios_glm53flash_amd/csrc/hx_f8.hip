// hx_f8.hip -- linear, and gate and up projections with their activation, over weights in 8-bit blocks (hx_f8.hpp) on gfx950.
//
//   y[m][n] = sum over blocks b of 128 k:  xs[m][b] ws[n / 128][b] sum over k in b: x[m][k] w[n][k]
//
// Lane 16 g + c of a matrix instruction holds a part of row c of either operand.  Which k that part is, is free as long as both operands
// agree: of a block of 128 k lane group g takes the 16-byte pieces g and 4 + g, which are consecutive over the lane groups in memory.
//
// The codes become fp16 (no rounding) for v_mfma_f32_16x16x32_f16, so that products are exact and their sums fp32.  (v_mfma_f32_16x16x128_f8f6f4
// adds 8 consecutive k after shifting each product to the largest exponent among them and drops what lies 2^13 and more below: 1.6e-5
// of the result, rms.)
#include "hx_f8.hpp"
#include "hx_kernels.hpp"

namespace hx {

namespace {

typedef uint32_t f8_u4 __attribute__((ext_vector_type(4)));

// Operand of 8 k from 8 codes.
HX_INLINE hx_h8 f8_half8(uint32_t lo, uint32_t hi)
{
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return hx_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's part of a block of a row: codes as loaded, or their fp16 values.
struct F8Raw {
    f8_u4 p[2];
};
struct F8Half {
    hx_h8 k[4];
};
HX_INLINE F8Half f8_half(const F8Raw& r)
{
    return {{f8_half8(r.p[0][0], r.p[0][1]), f8_half8(r.p[0][2], r.p[0][3]), f8_half8(r.p[1][0], r.p[1][1]), f8_half8(r.p[1][2], r.p[1][3])}};
}


// Lane group g's part of block b of a row (null: zeros).
HX_INLINE F8Half f8_operand(const uint8_t* row, int b, int g, int K)
{
    F8Raw v{};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = b * F8_BLOCK + 16 * (4 * h + g);
        if (row && k < K) v.p[h] = *reinterpret_cast<const f8_u4*>(row + k);
    }
    return f8_half(v);
}

// Products of 16 weight rows from n0 and 16 input rows from m0.
HX_INLINE hx_f4 f8_tile16(const uint8_t* x, const float* xs, const F8Blocks& w, int n0, int m0, int M, int N, int K)
{
    const int col = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, kb = (K + F8_BLOCK - 1) / F8_BLOCK;
    const uint8_t* wr = n0 + col < N ? w.codes + (size_t)(n0 + col) * K : nullptr;
    const uint8_t* xr = m0 + col < M ? x + (size_t)(m0 + col) * K : nullptr;
    const float* ws = w.scales + (size_t)(min(n0, N - 1) / F8_BLOCK) * kb;
    const float* s = xs + (size_t)min(m0 + col, M - 1) * kb;
    hx_f4 acc{0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < kb; ++b) {
        const F8Half wv = f8_operand(wr, b, g, K), xv = f8_operand(xr, b, g, K);
        hx_f4 p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv.k[j], xv.k[j], p, 0, 0, 0);
        const float f = s[b] * ws[b];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(f, p[e], acc[e]);
    }
    return acc;
}

HX_INLINE float f8_gated(float g, float u, float limit)
{
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
    return g / (1.0f + __expf(-g)) * u;
}

}  // namespace

__global__ __launch_bounds__(64) void f8_gemm_kernel(const uint8_t* x, const float* xs, F8Blocks w, void* y, int M, int N, int K,
                                                     bool y_fp32)
{
    const int n0 = 16 * blockIdx.x, lane = threadIdx.x;
    for (int m0 = 16 * blockIdx.y; m0 < M; m0 += 16 * gridDim.y) {
        const hx_f4 v = f8_tile16(x, xs, w, n0, m0, M, N, K);
        const int m = m0 + (lane & 15), n = n0 + 4 * (lane >> 4);
        if (m < M)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < N) {
                    const size_t i = (size_t)m * N + n + e;
                    if (y_fp32) static_cast<float*>(y)[i] = v[e];
                    else static_cast<_Float16*>(y)[i] = (_Float16)v[e];
                }
    }
}

__global__ __launch_bounds__(512) void f8_gate_up_kernel(const uint8_t* x, const float* xs, F8Blocks gate, F8Blocks up, uint8_t* q,
                                                         float* scales, int M, int N, int K, float limit)
{
    __shared__ uint32_t largest[8][16];
    const int block = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int n0 = block * F8_BLOCK + 16 * wave;
    for (int m0 = 16 * blockIdx.y; m0 < M; m0 += 16 * gridDim.y) {
        const hx_f4 g = f8_tile16(x, xs, gate, n0, m0, M, N, K), u = f8_tile16(x, xs, up, n0, m0, M, N, K);
        float v[4];
        uint32_t a = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = n0 + 4 * (lane >> 4) + e < N ? f8_gated(g[e], u[e], limit) : 0.0f;
            a = max(a, f8_abs_bits(v[e]));
        }
        a = max(a, (uint32_t)__shfl_xor((int)a, 16, 64));
        a = max(a, (uint32_t)__shfl_xor((int)a, 32, 64));
        if (lane < 16) largest[wave][lane] = a;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, largest[i][lane & 15]);
        const F8Scale s = f8_scale(a);
        const int m = m0 + (lane & 15), n = n0 + 4 * (lane >> 4);
        if (m < M) {
            if (n < N)  // N is a multiple of 16
                *reinterpret_cast<uint32_t*>(q + (size_t)m * N + n) = f8_codes(v[0] * s.factor, v[1] * s.factor, v[2] * s.factor, v[3] * s.factor);
            if (threadIdx.x < 16) scales[(size_t)m * ((N + F8_BLOCK - 1) / F8_BLOCK) + block] = s.scale;
        }
        __syncthreads();
    }
}

size_t f8_gemm_workspace_bytes(int, int, int) { return 0; }
size_t f8_gate_up_workspace_bytes(int, int, int) { return 0; }

hipError_t launch_f8_gemm(const uint8_t* x, const float* xs, const F8Blocks& w, void* y, int M, int N, int K, bool y_fp32, void*, size_t,
                          hipStream_t st)
{
    const int rows = M < 16 * 4096 ? (M + 15) / 16 : 4096;
    hipLaunchKernelGGL(f8_gemm_kernel, dim3((N + 15) / 16, rows < (1 << 26) / ((N + 15) / 16) + 1 ? rows : 1), dim3(64), 0, st, x, xs, w, y, M, N, K, y_fp32);
    return hipGetLastError();
}

hipError_t launch_f8_gate_up(const uint8_t* x, const float* xs, const F8Blocks& gate, const F8Blocks& up, uint8_t* q, float* scales,
                             int M, int N, int K, float limit, void*, size_t, hipStream_t st)
{
    hipLaunchKernelGGL(f8_gate_up_kernel, dim3((N + F8_BLOCK - 1) / F8_BLOCK, N < (1 << 20) && M > 16 ? (M < 256 ? (M + 15) / 16 : 16) : 1), dim3(512), 0, st,
                       x, xs, gate, up, q, scales, M, N, K, limit);
    return hipGetLastError();
}

}  // namespace hx
