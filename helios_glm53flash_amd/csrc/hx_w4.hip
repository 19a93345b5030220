// hx_w4.hip -- linear and row lookup over 4-bit weights with group scales (no trellis, no Hadamard) on gfx950.
//
//   weight (n, k) = scales[n][k / group] * (q(n, k) - zeros[n][k / group]),  q in 0..15, zeros 8 where there are none
//
// Words: row n is ceil(K / 128) blocks of 16 uint32; word 4 g + j of a block holds the octet of weights
// k = 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7), nibble 0 (the low bits) first.  So (word >> 4 p) & 0x000f000f is the pair
// k = 2p, 2p + 1 of the octet, and the 16 bytes that a lane loads (words 4 g .. 4 g + 3) are its operands of four
// consecutive 32-k matrix instructions (lane group g of each holds 8 consecutive k): no group of 32 k and more spans two
// instructions, whatever its size.
//
//   M <= 64  w4_rows_kernel: the waves of a workgroup split K and keep their part of x in registers; they walk over the
//            weight rows, every word read once, and add their sums through LDS.
//   M > 64   w4_tile_kernel: tiles of 128 (or 64) x 128 outputs, x through LDS, the words straight into operands.
#include "hx_mfma.hpp"
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

// The same as a matrix operand: a nibble put into the mantissa of 1024 (its low bits) or of 64 (bits 4..7) gives 1024 + q
// or 64 + q, and subtracting 1024 + zero or 64 + zero is exact (zero <= 255).  9 VALU instructions for 8 weights.
struct ZeroPair {
    hx_h2 lo, hi;  // 1024 + zero, 64 + zero
};
HX_INLINE ZeroPair zero_pair(uint32_t zero)
{
    const hx_h2 lo = u32_as_h2(zero * 0x00010001u + 0x64006400u);
    return {lo, lo - u32_as_h2(0x63806380u)};  // 960
}
HX_INLINE hx_h8 word_operand(uint32_t w, ZeroPair z)
{
    const uint32_t w8 = w >> 8;
    union {
        hx_h2 p[4];
        hx_h8 v;
    } o;
    o.p[0] = u32_as_h2((w & 0x000f000fu) | 0x64006400u) - z.lo;
    o.p[1] = u32_as_h2((w & 0x00f000f0u) | 0x54005400u) - z.hi;
    o.p[2] = u32_as_h2((w8 & 0x000f000fu) | 0x64006400u) - z.lo;
    o.p[3] = u32_as_h2((w8 & 0x00f000f0u) | 0x54005400u) - z.hi;
    return o.v;
}

// Scales (fp16, one per 16 bits) and zero points (one per 8 bits) of a block of 128 k, lowest group first.  GS: groups in a
// block, 1 where the group is 128 or longer.
template <int GS>
struct BlockScale {
    uint64_t s;
    uint32_t z;
    HX_INLINE float scale(int g) const { return (float)u16_as_h((uint16_t)(s >> (16 * g))); }
    HX_INLINE ZeroPair zero(int g) const { return zero_pair((z >> (8 * g)) & 255u); }
};

// Of block blk of row `row` (both inside the matrix).  A short last block reads the GS groups that end with the row and shifts
// them down, so groups past K have scale 0; a row of fewer than GS groups reads them one by one.
template <int GS, bool Z>
HX_INLINE BlockScale<GS> block_scale(const W4Args& a, size_t row, int blk)
{
    typedef uint32_t u32a2 __attribute__((aligned(2)));
    typedef uint64_t u64a2 __attribute__((aligned(2)));
    typedef uint16_t u16a1 __attribute__((aligned(1)));
    typedef uint32_t u32a1 __attribute__((aligned(1)));
    BlockScale<GS> r{0, 0};
    if constexpr (GS == 1) {
        const size_t i = row * a.groups + ((blk * 128) >> a.group_log2);
        r.s = h_as_u16(a.scales[i]);
        if constexpr (Z) r.z = a.zeros[i];
    } else {
        const int g0 = blk * GS;
        const _Float16* s = a.scales + row * a.groups;
        const uint8_t* z = a.zeros + row * a.groups;
        if (a.groups >= GS) {
            const int g = min(g0, a.groups - GS), off = g0 - g;
            if constexpr (GS == 2) r.s = *reinterpret_cast<const u32a2*>(s + g);
            else r.s = *reinterpret_cast<const u64a2*>(s + g);
            r.s >>= 16 * off;
            if constexpr (Z) {
                if constexpr (GS == 2) r.z = *reinterpret_cast<const u16a1*>(z + g);
                else r.z = *reinterpret_cast<const u32a1*>(z + g);
                r.z >>= 8 * off;
            }
        } else {
            for (int g = g0; g < a.groups; ++g) {
                r.s |= (uint64_t)h_as_u16(s[g]) << (16 * (g - g0));
                if constexpr (Z) r.z |= (uint32_t)z[g] << (8 * (g - g0));
            }
        }
    }
    if constexpr (!Z) r.z = 0x08080808u;
    return r;
}

HX_INLINE void store_y(void* y, size_t i, float v, bool y_fp32)
{
    if (y_fp32) static_cast<float*>(y)[i] = v;
    else static_cast<_Float16*>(y)[i] = (_Float16)v;
}

}  // namespace

// ---- M <= 64
//
// One wave load covers 16 / S weight rows over S consecutive blocks of 128 k (S * 64 bytes of each row): column n = s R + r of
// the matrix instruction is row r (R = 16 / S), block s, and row a = s R + t of the other operand is token t's x in block s.  Of
// the products those with equal s are wanted; for few tokens the unused rows so buy whole cache lines per row and four times
// as many rows to spread over the chip.  S = 4 serves 4 tokens, 2 serves 8, 1 serves 16 MT.
// A wave owns NS spans (S blocks each) of every WK NS, keeps x for them in registers and goes over tiles of NT R rows; each word
// is replaced by the next tile's as soon as it is decoded.  Per group the products are summed by the matrix
// instructions from zero, then scaled into the fp32 sums.
template <int S, int MT, int NS, int NT, int GS, bool Z>
__global__ __launch_bounds__(512) void w4_rows_kernel(const _Float16* x, W4Args a, void* y, int M, bool y_fp32, int wk)
{
    constexpr int R = 16 / S, H = 4 / S, SLOTS = 16 * H;  // rows of a load; 4-token pieces of a column; pieces kept per tile
    __shared__ hx_f4 red[2][8][NT * MT][SLOTS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave & (wk - 1), rw = wave / wk, wr = 8 / wk;  // the wave's place in K and in rows
    const int col = lane & 15, kg = lane >> 4, s = col / R, r = col % R;
    const int nb = (a.K + 127) / 128, nkb = ((nb + S - 1) / S + wk * NS - 1) / (wk * NS);  // blocks; rounds over K
    const int row_bytes = nb * 64, rows_wg = wr * NT * R;
    const int tiles = (a.N + rows_wg - 1) / rows_wg;

    hx_h8 xa[NS][MT][4];
    auto load_x = [&](int kb) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int blk = ((kb * NS + i) * wk + kw) * S + s;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int t = 16 * m + r;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = blk * 128 + 32 * j + 8 * kg;
                    xa[i][m][j] = hx_h8{};
                    if (t < M && k < a.K) xa[i][m][j] = *reinterpret_cast<const hx_h8*>(x + (size_t)t * a.K + k);
                }
            }
        }
    };
    hx_u4 w[NS][NT];
    BlockScale<GS> sc[NS][NT];
    auto load_w = [&](int i, int n, int tile, int kb) {
        const int row0 = (tile * wr + rw) * NT * R;
        const int blk = ((kb * NS + i) * wk + kw) * S + s, bc = min(blk, nb - 1);
        const size_t row = min(row0 + n * R + r, a.N - 1);
        w[i][n] = *reinterpret_cast<const hx_u4*>(reinterpret_cast<const char*>(a.words) + row * row_bytes + bc * 64 + kg * 16);
        sc[i][n] = block_scale<GS, Z>(a, row, bc);
        if (blk != bc) sc[i][n].s = 0;
    };
    load_x(0);
    int tile = blockIdx.x;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) load_w(i, n, tile, 0);
    int buf = 0;
    for (; tile < tiles; tile += gridDim.x, buf ^= 1) {
        hx_f4 acc[NT][MT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[n][m] = hx_f4{0.f, 0.f, 0.f, 0.f};
        for (int kb = 0; kb < nkb; ++kb) {
            if (nkb > 1) load_x(kb);
            const bool wrap = kb + 1 == nkb;
            const int next_tile = wrap ? min(tile + (int)gridDim.x, tiles - 1) : tile, next_kb = wrap ? 0 : kb + 1;
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const hx_u4 wv = w[i][n];
                    const BlockScale<GS> sv = sc[i][n];
                    hx_h8 b[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) b[j] = word_operand(wv[j], sv.zero(j * GS / 4));
                    load_w(i, n, next_tile, next_kb);
#pragma unroll
                    for (int g = 0; g < GS; ++g) {
                        const float f = sv.scale(g);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            hx_f4 c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int j = g * 4 / GS; j < (g + 1) * 4 / GS; ++j)
                                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[i][m][j], b[j], c, 0, 0, 0);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[n][m][e] = __builtin_fmaf(f, c[e], acc[n][m][e]);
                        }
                    }
                }
        }
        // lane: column col, rows 4 kg + e of the products; wanted where their blocks agree
        if (kg / H == s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) red[buf][wave][n * MT + m][col * H + kg % H] = acc[n][m];
        __syncthreads();  // the other buffer was read before the previous tile's barrier
        constexpr int ITEMS = NT * MT * R * H;  // pieces of 4 tokens of one row, per row part of the workgroup
        for (int i = threadIdx.x; i < ITEMS * wr; i += 512) {
            const int part = i / ITEMS, q = i % ITEMS;
            const int h = q % H, rr = q / H % R, m = q / H / R % MT, n = q / H / R / MT;
            hx_f4 v{0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < wk; ++k)
#pragma unroll
                for (int ss = 0; ss < S; ++ss) v += red[buf][part * wk + k][n * MT + m][(ss * R + rr) * H + h];
            const int row = (tile * wr + part) * NT * R + n * R + rr;
            if (row < a.N)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = 16 * m + 4 * h + e;
                    if (t < M) store_y(y, (size_t)t * a.N + row, v[e], y_fp32);
                }
        }
    }
}

// ---- M > 64
//
// A workgroup of 4 waves computes BM x 128 outputs; wave w the 32 columns (weight rows) 32 w.. for all BM rows.  x goes through a
// ring of LDS buffers of BM x 128 k, loaded by buffer loads with an LDS destination; 16-byte piece u of row m lies at
// piece u ^ (m & 15), so the 16 rows of a fragment read touch all banks.  The words go from memory into registers, PF chunks
// ahead, and become operands there: no wave decodes a weight another wave of the workgroup uses.
constexpr int W4T_BN = 128;

template <int BM, int GS, bool Z>
__device__ __forceinline__ void w4_tile(const _Float16* x, const W4Args& a, void* y, int M, bool y_fp32)
{
    constexpr int NBUF = 2, RB = BM / 16, NL = BM / 16;  // loads of 4 rows per wave: BM / 4 rows / 4 waves
    extern __shared__ __align__(16) _Float16 w4_lds[];   // [NBUF][BM][128]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, kg = lane >> 4;
    const int nb = (a.K + 127) / 128, row_bytes = nb * 64;
    const int mt = (M + BM - 1) / BM;
    const int m0 = (int)(blockIdx.x % mt) * BM, n0 = (int)(blockIdx.x / mt) * W4T_BN;
    const __amdgpu_buffer_rsrc_t rx = mf_rsrc(x + (size_t)m0 * a.K, (size_t)min(M - m0, BM) * a.K * sizeof(_Float16));
    int voff[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int r = 4 * (wave * NL + i) + (lane >> 4);  // rows past M (clamped) are computed but not stored
        voff[i] = (int)(((size_t)min(r, M - m0 - 1) * a.K + 8 * ((lane & 15) ^ (r & 15))) * sizeof(_Float16));
    }
    // past K a piece is the next row's or, past the end, zeros; its products are skipped below
    auto load_a = [&](int c) {
        _Float16* d = w4_lds + (size_t)(c % NBUF) * BM * 128 + wave * NL * 512;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(d + 512 * i), 16, voff[i],
                                                     c * 256, 0, 0);
    };
    size_t row[2];
    const char* wp[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        row[n] = min(n0 + 32 * wave + 16 * n + col, a.N - 1);
        wp[n] = reinterpret_cast<const char*>(a.words) + row[n] * row_bytes + kg * 16;
    }
    hx_f4 acc[RB][2];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[i][n] = hx_f4{0.f, 0.f, 0.f, 0.f};
    hx_u4 w[2];
    BlockScale<GS> sc[2];
    auto load_w = [&](int c) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            w[n] = *reinterpret_cast<const hx_u4*>(wp[n] + c * 64);
            sc[n] = block_scale<GS, Z>(a, row[n], c);
        }
    };
    load_a(0);
    load_w(0);
    for (int c = 0; c < nb; ++c) {
        __syncthreads();  // waits for this wave's loads of chunk c, then for the others'; buffer c + 1 is no longer read
        hx_h8 b[2][4];
        float f[2][GS];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) b[n][j] = word_operand(w[n][j], sc[n].zero(j * GS / 4));
#pragma unroll
            for (int g = 0; g < GS; ++g) f[n][g] = sc[n].scale(g);
        }
        if (c + 1 < nb) {
            load_a(c + 1);
            load_w(c + 1);
        }
        const _Float16* s = w4_lds + (size_t)(c % NBUF) * BM * 128;
        auto products = [&](int i, int nj) {
            hx_h8 xa[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                xa[j] = *reinterpret_cast<const hx_h8*>(s + (16 * i + col) * 128 + 8 * ((4 * j + kg) ^ col));
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int g = 0; g < GS; ++g) {
                    hx_f4 t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = g * 4 / GS; j < (g + 1) * 4 / GS; ++j)
                        if (j < nj) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[j], b[n][j], t, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][n][e] = __builtin_fmaf(f[n][g], t[e], acc[i][n][e]);
                }
        };
        const int nj = min(4, (a.K - 128 * c) / 32);
        if (nj == 4) {
#pragma unroll
            for (int i = 0; i < RB; ++i) products(i, 4);
        } else {
#pragma unroll
            for (int i = 0; i < RB; ++i) products(i, nj);
        }
    }
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int nn = n0 + 32 * wave + 16 * n + col;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = m0 + 16 * i + 4 * kg + e;
                if (m < M && nn < a.N) store_y(y, (size_t)m * a.N + nn, acc[i][n][e], y_fp32);
            }
        }
}

template <int BM, int GS, bool Z>
__global__ __launch_bounds__(256) void w4_tile_kernel(const _Float16* x, W4Args a, void* y, int M, bool y_fp32)
{
    w4_tile<BM, GS, Z>(x, a, y, M, y_fp32);
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

namespace {

struct W4Call {
    const _Float16* x;
    const W4Args& a;
    void* y;
    int M;
    bool y_fp32;
    hipStream_t st;
};

template <int S, int MT, int NS, int NT, int GS, bool Z>
hipError_t rows_launch(const W4Call& c)
{
    const int spans = ((c.a.K + 127) / 128 + S - 1) / S;
    int wk = 1;  // waves along K: as many as have spans, up to all 8
    while (wk < 8 && wk * NS < spans) wk *= 2;
    const int rows = 8 / wk * NT * 16 / S, tiles = (c.a.N + rows - 1) / rows;
    hipLaunchKernelGGL((w4_rows_kernel<S, MT, NS, NT, GS, Z>), dim3(tiles < 512 ? tiles : 512), dim3(512), 0, c.st, c.x, c.a,
                       c.y, c.M, c.y_fp32, wk);
    return hipGetLastError();
}

template <int BM, int GS, bool Z>
hipError_t tile_launch(const W4Call& c)
{
    constexpr size_t lds = sizeof(_Float16) * 2 * BM * 128;
    const long tiles = (long)((c.M + BM - 1) / BM) * ((c.a.N + W4T_BN - 1) / W4T_BN);
    hipLaunchKernelGGL((w4_tile_kernel<BM, GS, Z>), dim3((unsigned)tiles), dim3(256), lds, c.st, c.x, c.a, c.y, c.M, c.y_fp32);
    return hipGetLastError();
}

template <int GS, bool Z>
hipError_t gemm_launch(const W4Call& c)
{
    if (c.M <= 4) return rows_launch<4, 1, 2, 4, GS, Z>(c);
    if (c.M <= 8) return rows_launch<2, 1, 2, 4, GS, Z>(c);
    if (c.M <= 16) return rows_launch<1, 1, 4, 2, GS, Z>(c);
    if (c.M <= 32) return rows_launch<1, 2, 2, 2, GS, Z>(c);
    if (c.M <= 64) return rows_launch<1, 4, 1, 2, GS, Z>(c);
    return tile_launch<128, GS, Z>(c);
}

template <int GS>
hipError_t gemm_launch(const W4Call& c)
{
    return c.a.zeros ? gemm_launch<GS, true>(c) : gemm_launch<GS, false>(c);
}

}  // namespace

hipError_t launch_w4_gemm(const _Float16* x, const W4Args& a, void* y, int M, bool y_fp32, hipStream_t st)
{
    if (M <= 0 || a.N <= 0) return hipSuccess;
    const W4Call c{x, a, y, M, y_fp32, st};
    return a.group_log2 == 5 ? gemm_launch<4>(c) : a.group_log2 == 6 ? gemm_launch<2>(c) : gemm_launch<1>(c);
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
