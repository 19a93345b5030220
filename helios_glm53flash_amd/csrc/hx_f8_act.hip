// hx_f8_act.hip -- activations into 8-bit blocks (hx_f8.hpp) on gfx950: as they are, or behind the residual's addition and the
// root-mean-square norm.
//
// A thread holds octets of 8 consecutive values; the 16 octets of a block are in 16 consecutive lanes (a DPP row), which find the
// block's largest value among themselves.
#include "hx_f8.hpp"
#include "hx_kernels.hpp"

namespace hx {

namespace {

typedef float f8_v4 __attribute__((ext_vector_type(4)));

HX_INLINE void load8(const _Float16* p, float (&v)[8])
{
    const hx_h8 h = *reinterpret_cast<const hx_h8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}
HX_INLINE void load8(const float* p, float (&v)[8])
{
    const f8_v4 a = *reinterpret_cast<const f8_v4*>(p), b = *reinterpret_cast<const f8_v4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[i + 4] = b[i];
}
HX_INLINE void store8(_Float16* p, const float (&v)[8])
{
    hx_h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[i];
    *reinterpret_cast<hx_h8*>(p) = h;
}
HX_INLINE void store8(float* p, const float (&v)[8])
{
    *reinterpret_cast<f8_v4*>(p) = f8_v4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f8_v4*>(p + 4) = f8_v4{v[4], v[5], v[6], v[7]};
}

// Codes and scale of the block that 16 lanes hold (lanes past the row's end hold zeros and store nothing).  All lanes of a row of 16
// take part.
HX_INLINE void store_block(uint8_t* q, float* scale, int octet, bool live, const float (&v)[8])
{
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, f8_abs_bits(v[i]));
    const F8Scale s = f8_scale(f8_row_max(a));
    if (!live) return;
    const float f = s.factor;
    uint2 c;
    c.x = f8_codes(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
    c.y = f8_codes(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
    *reinterpret_cast<uint2*>(q) = c;
    if ((octet & 15) == 0) *scale = s.scale;
}

// The type that the sum is kept in.
template <typename T, typename R>
struct F8Kept {
    typedef R type;
};
template <typename T>
struct F8Kept<T, void> {
    typedef T type;
};

}  // namespace

template <typename T>
__global__ __launch_bounds__(256) void f8_quantize_kernel(const T* x, uint8_t* q, float* scales, uint32_t items, int K, long ld)
{
    const uint32_t kb = (uint32_t)(K + F8_BLOCK - 1) / F8_BLOCK;
    const uint32_t item = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= items) return;
    const uint32_t row = item / kb, block = item % kb;
    const int octet = (int)(block * 16 + (threadIdx.x & 15));
    const bool live = octet * 8 < K;
    float v[8] = {};
    if (live) load8(x + (size_t)row * ld + octet * 8, v);
    store_block(q + (size_t)row * K + octet * 8, scales + item, octet, live, v);
}

// One workgroup a row.  h = x + residual, rounded to the residual's type R and kept in `out` (R == void: h = x, kept nowhere); n =
// h rsqrt(mean h^2 + eps) weight, in fp32; y = fp16 n, q and scales its blocks.  OPT octets a thread stay in registers; OPT == 0 takes
// rows of any length and reads `out` (or x) again for the second half.
template <typename T, typename R, int OPT>
__global__ __launch_bounds__(OPT == 0 ? 1024 : 512) void f8_norm_kernel(F8NormArgs a)
{
    constexpr bool RES = !__is_same(R, void);
    using RT = typename F8Kept<T, R>::type;
    __shared__ float part[16];
    const size_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    const RT* res = static_cast<const RT*>(a.residual) + row * a.K;
    RT* out = static_cast<RT*>(a.out) + row * a.K;
    const int octets = a.K / 8, nt = (int)blockDim.x;

    auto sum8 = [&](int o, float (&v)[8]) {
        load8(x + 8 * o, v);
        if constexpr (RES) {
            float r[8];
            load8(res + 8 * o, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)(RT)(v[i] + r[i]);
        }
    };
    auto finish8 = [&](int o, bool live, float (&v)[8], const float (&w)[8], float r) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
        if (a.y && live) store8(static_cast<_Float16*>(a.y) + row * a.K + 8 * o, v);
        if (a.q)
            store_block(static_cast<uint8_t*>(a.q) + row * a.K + 8 * o,
                        a.scales + row * ((a.K + F8_BLOCK - 1) / F8_BLOCK) + o / 16, o, live, v);
    };
    auto weight8 = [&](int o, float (&w)[8]) {
        if (a.weight32) load8(static_cast<const float*>(a.weight) + 8 * o, w);
        else load8(static_cast<const _Float16*>(a.weight) + 8 * o, w);
    };
    auto square8 = [](const float (&v)[8]) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(v[i], v[i], s);
        return s;
    };
    // 1 / root of the mean square, from the threads' sums: lanes, then waves, always in the same order
    auto inverse = [&](float s) {
#pragma unroll
        for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m, 64);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        hx_lds_barrier();
        s = 0.0f;
        for (int w = 0; w < nt / 64; ++w) s += part[w];
        return 1.0f / __builtin_sqrtf(s / (float)a.K + a.eps);
    };

    float s = 0.0f;
    if constexpr (OPT > 0) {
        float v[OPT][8] = {}, w[OPT][8] = {};
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int o = (int)threadIdx.x + j * nt;
            if (o < octets) sum8(o, v[j]), weight8(o, w[j]);
        }
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int o = (int)threadIdx.x + j * nt;
            if (RES && o < octets) store8(out + 8 * o, v[j]);
            s += square8(v[j]);
        }
        const float r = inverse(s);
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int o = (int)threadIdx.x + j * nt;
            if ((o & ~15) < octets) finish8(o, o < octets, v[j], w[j], r);
        }
    } else {
        for (int o = (int)threadIdx.x; o < octets; o += nt) {
            float v[8];
            sum8(o, v);
            if constexpr (RES) store8(out + 8 * o, v);
            s += square8(v);
        }
        const float r = inverse(s);
        for (int o = (int)threadIdx.x; (o & ~15) < octets; o += nt) {
            float v[8] = {}, w[8] = {};
            if (o < octets) {
                if constexpr (RES) load8(out + 8 * o, v);
                else load8(x + 8 * o, v);
                weight8(o, w);
            }
            finish8(o, o < octets, v, w, r);
        }
    }
}

namespace {

constexpr size_t F8_NORM_ROWS = 1u << 21;  // of a launch: 2^31 threads

template <typename T, typename R>
void norm_launch(const F8NormArgs& a, int M, hipStream_t st)
{
    const int octets = a.K / 8;
    auto threads = [&](int per) { return ((octets + per - 1) / per + 63) / 64 * 64; };
    if (octets <= 512) hipLaunchKernelGGL((f8_norm_kernel<T, R, 1>), dim3(M), dim3(threads(1)), 0, st, a);
    else if (octets <= 1024) hipLaunchKernelGGL((f8_norm_kernel<T, R, 2>), dim3(M), dim3(threads(2)), 0, st, a);
    else if (octets <= 2048) hipLaunchKernelGGL((f8_norm_kernel<T, R, 4>), dim3(M), dim3(threads(4)), 0, st, a);
    else hipLaunchKernelGGL((f8_norm_kernel<T, R, 0>), dim3(M), dim3(1024), 0, st, a);
}

template <typename T>
void norm_launch(const F8NormArgs& a, int M, bool r32, hipStream_t st)
{
    if (!a.residual) norm_launch<T, void>(a, M, st);
    else if (r32) norm_launch<T, float>(a, M, st);
    else norm_launch<T, _Float16>(a, M, st);
}

}  // namespace

hipError_t launch_f8_norm(const F8NormArgs& a, int M, bool x32, bool r32, hipStream_t st)
{
    const size_t kb = (size_t)(a.K + F8_BLOCK - 1) / F8_BLOCK;
    auto behind = [](const void* p, size_t bytes) { return p ? static_cast<const char*>(p) + bytes : nullptr; };
    for (size_t m = 0; m < (size_t)M; m += F8_NORM_ROWS) {
        F8NormArgs c = a;
        c.x = behind(a.x, m * a.ld * (x32 ? 4 : 2));
        c.residual = behind(a.residual, m * a.K * (r32 ? 4 : 2));
        c.out = const_cast<char*>(behind(a.out, m * a.K * (r32 ? 4 : 2)));
        c.y = const_cast<char*>(behind(a.y, m * a.K * 2));
        c.q = const_cast<char*>(behind(a.q, m * a.K));
        if (a.scales) c.scales = a.scales + m * kb;
        const int rows = (int)((size_t)M - m < F8_NORM_ROWS ? (size_t)M - m : F8_NORM_ROWS);
        if (x32) norm_launch<float>(c, rows, r32, st);
        else norm_launch<_Float16>(c, rows, r32, st);
    }
    return hipGetLastError();
}

hipError_t launch_f8_quantize(const void* x, bool x32, uint8_t* q, float* scales, int M, int K, long ld, hipStream_t st)
{
    const int kb = (K + F8_BLOCK - 1) / F8_BLOCK, most = (int)((1u << 27) / kb);  // rows of a launch: 2^27 blocks, 2^31 threads
    for (long m = 0; m < M; m += most) {
        const uint32_t items = (uint32_t)(M - m < most ? M - m : most) * kb;
        const dim3 grid((items + 15) / 16);
        if (x32)
            hipLaunchKernelGGL((f8_quantize_kernel<float>), grid, dim3(256), 0, st, static_cast<const float*>(x) + m * ld, q + m * K,
                               scales + m * kb, items, K, ld);
        else
            hipLaunchKernelGGL((f8_quantize_kernel<_Float16>), grid, dim3(256), 0, st, static_cast<const _Float16*>(x) + m * ld,
                               q + m * K, scales + m * kb, items, K, ld);
    }
    return hipGetLastError();
}

}  // namespace hx
