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
//   M <= 8  w4_rows_kernel: the waves of a workgroup split K and keep their part of x in registers; they walk over the
//           weight rows, every word read once, and add their sums through LDS.
//   M > 8   w4_tile_kernel: tiles of 16 to 128 by 64 or 128 outputs, x through LDS, the words straight into operands.
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

// Buffer accesses return 0 beyond a descriptor's bytes (and beyond 2^30 always, which marks what must read as 0).  Everything
// that decides about that is in the per-lane offset.
constexpr int W4_NONE = 0x7ffffff0;
HX_INLINE __amdgpu_buffer_rsrc_t w4_rsrc(const void* base, long bytes, long most = 0x40000000l)
{
    return mf_rsrc(base, (size_t)(bytes < 0 ? 0 : bytes > most ? most : bytes));
}

// Scales (fp16) and zero points of a block of 128 k, lowest group first.  GS: groups in a block, 1 where the group is 128 or
// longer.  V: the GS groups of a block are one aligned piece (K a multiple of 128, aligned pointers); without, each group is
// loaded by itself.  Which of the two is not decided in the kernels: branches between the loads of a ring make the compiler
// wait for all of them.
template <int GS, bool Z, bool V>
struct BlockScale {
    static constexpr int NS = GS == 1 ? 1 : V ? GS / 2 : GS, NZ = GS == 1 || V ? 1 : GS;
    uint32_t s[NS], z[NZ];  // as loaded: converted where they are used, since anything earlier would wait for the load
    HX_INLINE float scale(int g) const
    {
        if constexpr (NS == GS) return (float)u16_as_h((uint16_t)s[g]);
        else return (float)u16_as_h((uint16_t)(s[g >> 1] >> (16 * (g & 1))));
    }
    HX_INLINE ZeroPair zero(int g) const
    {
        if constexpr (!Z) return {u32_as_h2(0x64086408u), u32_as_h2(0x54805480u)};  // 1032, 72
        else if constexpr (NZ == GS) return zero_pair(z[g]);
        else return zero_pair((z[0] >> (8 * g)) & 255u);
    }
};

// The scales of NT <= 4 columns' blocks are loaded together: lane group kg those of column kg, `first` that column's, or W4_NO_SCALE
// (zero points are read through descriptors of at most 2^29 bytes) in lane groups past NT; then every lane group gets all NT.
// A load whose lanes are in 16 rows takes the address unit 62 cycles with the row's value in all four lane groups (the words, 16
// bytes a lane, 33) and 19 in one; while each column had a load of its own, 5 rows of 8192 -> 4096 in groups of 32 took 10.5 us for 8.8.
constexpr int W4_NO_SCALE = 1 << 29;
template <int NT>
HX_INLINE void spread(uint32_t v, uint32_t (&o)[NT])
{
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);  // columns 0 1 0 1 | 2 3 2 3 by lane group
    const auto a = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false);
    o[0] = a[0];
    if constexpr (NT > 1) o[1] = a[1];
    if constexpr (NT > 2) {
        const auto b = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
        o[2] = b[0];
        if constexpr (NT > 3) o[3] = b[1];
    }
}
template <int NT, int GS, bool Z, bool V>
HX_INLINE void spread_scale(const BlockScale<GS, Z, V>& v, BlockScale<GS, Z, V> (&o)[NT])
{
    uint32_t t[NT];
    if constexpr (GS == 1 && Z) {
        spread<NT>(v.s[0] | v.z[0] << 16, t);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n].s[0] = t[n], o[n].z[0] = t[n] >> 16;
    } else {
#pragma unroll
        for (int i = 0; i < BlockScale<GS, Z, V>::NS; ++i) {
            spread<NT>(v.s[i], t);
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n].s[i] = t[n];
        }
        if constexpr (Z)
#pragma unroll
            for (int i = 0; i < BlockScale<GS, Z, V>::NZ; ++i) {
                spread<NT>(v.z[i], t);
#pragma unroll
                for (int n = 0; n < NT; ++n) o[n].z[i] = t[n];
            }
    }
}

// Of block blk of the row whose first group lies `first` groups behind the descriptors' base.  Groups past K, and rows past the
// descriptors, have scale 0.
template <int GS, bool Z, bool V>
HX_INLINE BlockScale<GS, Z, V> block_scale(__amdgpu_buffer_rsrc_t rs, __amdgpu_buffer_rsrc_t rz, const W4Args& a, int first,
                                           int blk)
{
    BlockScale<GS, Z, V> r;
    if constexpr (GS == 1) {
        const int g = (blk * 128) >> a.group_log2, i = g < a.groups ? first + g : W4_NONE >> 1;
        r.s[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, 2 * i, 0, 0);
        if constexpr (Z) r.z[0] = __builtin_amdgcn_raw_buffer_load_b8(rz, i, 0, 0);
    } else if constexpr (V) {
        const int i = blk * GS < a.groups ? first + blk * GS : W4_NONE >> 1;
        if constexpr (GS == 2) {
            r.s[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, 2 * i, 0, 0);
            if constexpr (Z) r.z[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rz, i, 0, 0);
        } else {
            const auto v = __builtin_amdgcn_raw_buffer_load_b64(rs, 2 * i, 0, 0);
            r.s[0] = v[0], r.s[1] = v[1];
            if constexpr (Z) r.z[0] = __builtin_amdgcn_raw_buffer_load_b32(rz, i, 0, 0);
        }
    } else {
#pragma unroll
        for (int g = 0; g < GS; ++g) {
            const int i = blk * GS + g < a.groups ? first + blk * GS + g : W4_NONE >> 1;
            r.s[g] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, 2 * i, 0, 0);
            if constexpr (Z) r.z[g] = __builtin_amdgcn_raw_buffer_load_b8(rz, i, 0, 0);
        }
    }
    return r;
}

HX_INLINE void store_y(void* y, size_t i, float v, bool y_fp32)
{
    if (y_fp32) static_cast<float*>(y)[i] = v;
    else static_cast<_Float16*>(y)[i] = (_Float16)v;
}

}  // namespace

// ---- up to 8 rows
//
// One wave load covers 16 / S weight rows over S consecutive blocks of 128 k (S * 64 bytes of each row): column n = s R + r of
// the matrix instruction is row r (R = 16 / S), block s, and row a = s R + t of the other operand is token t's x in block s.  Of
// the products those with equal s are wanted; for few tokens the unused rows so buy whole cache lines per row and four times
// as many rows to spread over the chip.  S = 4 serves 4 tokens, 2 serves 8.
// A wave owns NS spans (S blocks each) of every WK NS, keeps x for them in registers and goes over tiles of NT R rows; each word
// is replaced by the next tile's as soon as it is decoded.  Per group the products are summed by the matrix
// instructions from zero, then scaled into the fp32 sums.
// Bound by memory where the weights are many: 8 rows of 4096 -> 151552 in groups of 128 take 66 us, 4.9 TB/s (a copy of 4 GiB runs at 4.8).
// Of the 8.0 us of one row of 4096 -> 12288 (26 MB, 5.4 us) and the 8.8 of five of 8192 -> 4096 in groups of 32 (20 MB, 4.2 us) about
// 4 are launch and the first load's latency, which a call of 4 MB also takes.
template <int S, int WAVES, int NS, int NT, int GS, bool Z, bool V>
__device__ __forceinline__ void w4_rows(const _Float16* x, const W4Args& a, void* y, int M, bool y_fp32, int wk)
{
    constexpr int R = 16 / S, H = 4 / S;  // rows of a load; 4-token pieces of a column
    __shared__ float red[WAVES][NT][4 * H][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave & (wk - 1), rw = wave / wk, wr = WAVES / wk;  // the wave's place in K and in rows
    const int col = lane & 15, kg = lane >> 4, s = col / R, r = col % R;
    const int nb = (a.K + 127) / 128, nkb = ((nb + S - 1) / S + wk * NS - 1) / (wk * NS);  // blocks; rounds over K
    const int row_bytes = nb * 64, rows_wg = wr * NT * R;
    const int tiles = (a.N + rows_wg - 1) / rows_wg;

    const __amdgpu_buffer_rsrc_t rx = w4_rsrc(x, (long)M * a.K * 2);
    hx_h8 xa[NS][4];
    auto load_x = [&](int kb) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int k = (((kb * NS + i) * wk + kw) * S + s) * 128 + 8 * kg;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int off = k + 32 * j < a.K ? (r * a.K + k + 32 * j) * 2 : W4_NONE;
                xa[i][j] = __builtin_bit_cast(hx_h8, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 0, 0));
            }
        }
    };
    hx_u4 w[NS][NT];
    BlockScale<GS, Z, V> sc[NS];
    __amdgpu_buffer_rsrc_t rw_, rs, rz;
    auto aim = [&](int tile) {  // descriptors of the tile's rows (nothing left of the matrix: every load is 0)
        const long row0 = (long)(tile * wr + rw) * NT * R, left = tile < tiles ? a.N - row0 : 0;
        rw_ = w4_rsrc(reinterpret_cast<const char*>(a.words) + row0 * row_bytes, left * row_bytes);
        rs = w4_rsrc(a.scales + row0 * a.groups, left * a.groups * 2);
        rz = w4_rsrc(Z ? a.zeros + row0 * a.groups : nullptr, Z ? left * a.groups : 0, W4_NO_SCALE);
    };
    const int lane_off = r * row_bytes + s * 64 + kg * 16, lane_group = kg < NT ? (kg * R + r) * a.groups : W4_NO_SCALE;
    auto load_w = [&](int i, int n, int kb) {
        const int span = (kb * NS + i) * wk + kw;
        // a block past K reads the next row's words: x is 0 there, and the scale
        w[i][n] = __builtin_bit_cast(hx_u4, __builtin_amdgcn_raw_buffer_load_b128(rw_, lane_off + n * R * row_bytes + span * (S * 64), 0, 0));
        if (n == 0) sc[i] = block_scale<GS, Z, V>(rs, rz, a, lane_group, span * S + s);
    };
    int tile = blockIdx.x;
    aim(tile);
    load_x(0);
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) load_w(i, n, 0);
    for (; tile < tiles; tile += gridDim.x) {
        hx_f4 acc[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n] = hx_f4{0.f, 0.f, 0.f, 0.f};
        for (int kb = 0; kb < nkb; ++kb) {
            if (nkb > 1) load_x(kb);
            const bool wrap = kb + 1 == nkb;
            const int next_kb = wrap ? 0 : kb + 1;
            if (wrap) aim(tile + gridDim.x);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                BlockScale<GS, Z, V> all[NT];
                spread_scale<NT>(sc[i], all);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const hx_u4 wv = w[i][n];
                    const BlockScale<GS, Z, V> sv = all[n];
                    hx_h8 b[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) b[j] = word_operand(wv[j], sv.zero(j * GS / 4));
                    load_w(i, n, next_kb);
                    // the loads stay here, ahead of this word's products: sunk to the end of the tile they cost 10 % of a long walk
                    // (4096 -> 151552, 1 row: 65 -> 59 us)
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int g = 0; g < GS; ++g) {
                        const float f = sv.scale(g);
                        hx_f4 c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = g * 4 / GS; j < (g + 1) * 4 / GS; ++j)
                            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[i][j], b[j], c, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[n][e] = __builtin_fmaf(f, c[e], acc[n][e]);
                    }
                }
            }
        }
        // lane: column col, rows 4 kg + e of the products; wanted where their blocks agree
        if (kg / H == s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) red[wave][n][kg % H * 4 + e][col] = acc[n][e];
        hx_lds_barrier();
        constexpr int ITEMS = NT * 4 * H * R;  // outputs per row part of the workgroup
        for (int i = threadIdx.x; i < ITEMS * wr; i += 64 * WAVES) {
            const int part = i / ITEMS, q = i % ITEMS, rr = q % R, t = q / R % (4 * H), n = q / R / (4 * H);
            const int row = (tile * wr + part) * NT * R + n * R + rr;
            float v = 0.0f;
            for (int k = 0; k < wk; ++k)
#pragma unroll
                for (int ss = 0; ss < S; ++ss) v += red[part * wk + k][n][t][ss * R + rr];
            if (row < a.N && t < M) store_y(y, (size_t)t * a.N + row, v, y_fp32);
        }
        hx_lds_barrier();  // the sums are read before the next tile's overwrite them
    }
}

template <int S, int WAVES, int NS, int NT, int GS, bool Z, bool V>
__global__ __launch_bounds__(64 * WAVES) void w4_rows_kernel(const _Float16* x, W4Args a, void* y, int M, bool y_fp32, int wk)
{
    w4_rows<S, WAVES, NS, NT, GS, Z, V>(x, a, y, M, y_fp32, wk);
}

// ---- more rows
//
// A workgroup computes BM x 64 NT outputs; its waves are KS parts of K by four column groups of 16 NT weight rows.  A step takes
// KS consecutive blocks of 128 k, one for each part.  x goes through a ring of PF LDS stages [KS][BM][128], filled by buffer loads
// with an LDS destination (256 consecutive bytes of a row); 16-byte piece u of row m lies at piece u ^ (m & 15), so the 16
// rows of a fragment read touch all banks.  The words go from memory into registers, as many steps ahead, and become operands
// there: no wave decodes a weight that another wave of the workgroup uses.
// With few rows the address unit is the busiest, by its counter 70 % of the time: of the 1900 cycles of a step of 64 x 64 outputs by 256 k in
// groups of 64, x takes 512, the words 264, scales and zero points 248, which is 54 %; the rest it holds requests that wait.  The VALU
// is busy half as much: 45 rows of 4096 -> 12288 15.6 us, 29 MB.  With many it is the
// matrix instructions at what clock the power limit leaves (1.7 GHz, 52 % busy): 2000 rows of 4096 -> 24576 in groups of 128
// 382 to 396 us, 1.02 to 1.05 PFLOP/s, where the library's fp16 product of 8192^3 runs at 1.26.  Groups of 32 have four products to scale where
// those have one: the same with zero points 510 us, vector instructions in 69 % of the cycles (53) and the matrix pipe in 37 % (54).
struct W4Split {
    int splits, steps;  // workgroups that share a tile's K, steps of each
    hx_f4* partial;     // [tiles][splits][RB][NT][4][64]
    int* counters;      // arrivals per tile, zero between calls
};

template <int BM, int NT, int KS, int PF, int GS, bool Z, bool V>
__device__ __forceinline__ void w4_tile(const _Float16* x, const W4Args& a, void* y, int M, bool y_fp32, W4Split sp)
{
    constexpr int RB = BM / 16, NL = BM / 16;  // row blocks; x loads (4 rows each) of a wave per step
    // vector memory instructions of a wave: per step, and for the scales of every SP-th
    constexpr int NVM = NL + NT, NSC = (V || GS == 1 ? 1 : GS) * (Z ? 2 : 1), SP = 4 / NT;
    static_assert(PF % SP == 0);
    extern __shared__ __align__(16) _Float16 w4_lds[];  // [PF][KS][BM][128]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave >> 2, cw = wave & 3, col = lane & 15, kg = lane >> 4;
    const int nb = (a.K + 127) / 128, row_bytes = nb * 64;
    const int tile = (int)(blockIdx.x / sp.splits), split = (int)(blockIdx.x % sp.splits);
    const int first = split * sp.steps, steps = min(first + sp.steps, (nb + KS - 1) / KS);  // this split's steps
    const int mt = (M + BM - 1) / BM;
    // Workgroups go to the 8 XCDs in turn.  While x fits an XCD's L2, the row tiles of a column group stay on one, which then reads the
    // words once (512 rows of 4096 -> 12288 69.3 -> 66.4 us, 256 rows 42.4 -> 40.7); beyond, row tiles in turn leave each XCD a
    // part of x (2000 rows 195 us against 203, 4096 rows of 4096 -> 4096 132 against 149).
    const int mine = (a.N + 64 * NT - 1) / (64 * NT) / 8 * 8 * mt;  // tiles of whole groups of 8 columns
    const bool xcd = sp.splits == 1 && tile < mine && (long)M * a.K <= 1l << 21;
    const int m0 = (xcd ? (tile >> 3) % mt : tile % mt) * BM, n0 = (xcd ? (tile >> 3) / mt * 8 + (tile & 7) : tile / mt) * (64 * NT);
    const long left = min(a.N - n0, 64 * NT);
    const char *xb = reinterpret_cast<const char*>(x + (size_t)m0 * a.K), *wb = reinterpret_cast<const char*>(a.words) + (size_t)n0 * row_bytes;
    const int x_bytes = min(M - m0, BM) * a.K * 2, w_bytes = (int)left * row_bytes;
    // From byte `at` on; nothing from step `steps` on.  The lanes' offsets are the same in all steps, and nothing branches.
    auto stepped = [&](const char* base, int at, int bytes, int c) {
        return mf_rsrc(base + at, (size_t)(max(bytes - at, 0) & ((c - steps) >> 31)));
    };
    const __amdgpu_buffer_rsrc_t rs = w4_rsrc(a.scales + (size_t)n0 * a.groups, left * a.groups * 2);
    const __amdgpu_buffer_rsrc_t rz = w4_rsrc(Z ? a.zeros + (size_t)n0 * a.groups : nullptr, Z ? left * a.groups : 0, W4_NO_SCALE);
    // rows past M and pieces past K hold anything: the former are not stored, the products of the latter are skipped
    int xoff[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int r = 4 * (cw * NL + i) + (lane >> 4);
        xoff[i] = (r * a.K + 8 * ((lane & 15) ^ (r & 15))) * 2;
    }
    auto load_x = [&](int i, int slot, int c) {
        _Float16* d = w4_lds + (slot * KS + part) * (BM * 128) + cw * NL * 512;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(stepped(xb, (c * KS + part) * 256, x_bytes, c),
                                                 (__attribute__((address_space(3))) void*)(d + 512 * i), 16, xoff[i], 0, 0, 0);
    };
    hx_u4 w[PF][NT];
    BlockScale<GS, Z, V> sc;
    const int lane_group = (16 * (cw * NT + kg % NT) + col) * a.groups;
    auto load_scales = [&](int c) {  // of steps c .. c + SP - 1: lane group kg takes column kg % NT, step c + kg / NT
        sc = block_scale<GS, Z, V>(rs, rz, a, lane_group, (c + kg / NT) * KS + part);
        asm volatile("" ::: "memory");
    };
    auto load_w = [&](int slot, int c) {
        const __amdgpu_buffer_rsrc_t rw = stepped(wb, (c * KS + part) * 64, w_bytes, c);
#pragma unroll
        for (int n = 0; n < NT; ++n)
            w[slot][n] = __builtin_bit_cast(
                hx_u4, __builtin_amdgcn_raw_buffer_load_b128(rw, (16 * (cw * NT + n) + col) * row_bytes + kg * 16, 0, 0));
    };
    hx_f4 acc[RB][NT];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[i][n] = hx_f4{0.f, 0.f, 0.f, 0.f};
    // The waits below, and the compiler's, count a step's loads: steps stay apart, the words come first in each, and every step
    // issues its loads, past the end as accesses that touch no memory (where they depended on the step, each use of the words
    // waited for all loads in flight: 13 us instead of x at 16 rows of 4096 -> 2048).
    if constexpr (SP >= PF) load_scales(first);
#pragma unroll
    for (int u = 0; u < PF - 1; ++u) {
        asm volatile("" ::: "memory");
        if ((u + 1) % SP == 0 && u + 1 == PF - SP) load_scales(first);
        load_w(u, first + u);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < NL; ++i) load_x(i, u, first + u);
    }
    BlockScale<GS, Z, V> sv[4];  // of SP steps
    auto step = [&](auto slot, int c, bool whole) {
        constexpr int u = decltype(slot)::value;
        // the decode of a later step's words would wait for their loads here
        __builtin_amdgcn_sched_barrier(0);
        // x of step c has arrived once at most what the PF - 2 steps before this one have loaded is outstanding
        constexpr int later = [] {
            int n = 0;
            for (int d = 1; d <= PF - 2; ++d) n += NVM + ((u + PF - d) % SP == 0 ? NSC : 0);
            return n;
        }();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(qt_vmcnt(later));
        hx_lds_barrier();  // and the other waves'; the stage of step c - 1 is no longer read
        hx_h8 b[NT][4];
        float f[NT][GS];
        if constexpr (u % SP == 0) spread_scale<4>(sc, sv);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const BlockScale<GS, Z, V>& s = sv[u % SP * NT + n];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[n][j] = word_operand(w[u][n][j], s.zero(j * GS / 4));
#pragma unroll
            for (int g = 0; g < GS; ++g) f[n][g] = s.scale(g);
        }
        asm volatile("" ::: "memory");
        if constexpr (u % SP == 0) load_scales(c + SP);
        load_w((u + PF - 1) % PF, c + PF - 1);
        asm volatile("" ::: "memory");
        const _Float16* s = w4_lds + (u * KS + part) * (BM * 128);
        const int left_k = whole ? 128 : a.K - 128 * (c * KS + part);  // of K in this block
        hx_h8 xa[2][4];
        auto fragment = [&](int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                xa[i & 1][j] = *reinterpret_cast<const hx_h8*>(s + (16 * i + col) * 128 + 8 * ((4 * j + kg) ^ col));
        };
        fragment(0);
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            // One row block's products, the next one's fragments and one x load at a time (2000 rows 412 -> 405 us against all x
            // loads at the start of a step; few rows the same).
            __builtin_amdgcn_sched_barrier(0);
            load_x(i, (u + PF - 1) % PF, c + PF - 1);
            if (i + 1 < RB) fragment(i + 1);
            if (!whole)  // what lies behind a row's K, x of another row or nothing, counts as 0 (as do the scales there)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (32 * j >= left_k) xa[i & 1][j] = hx_h8{};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int g = 0; g < GS; ++g) {
                    hx_f4 t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = g * 4 / GS; j < (g + 1) * 4 / GS; ++j)
                        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(xa[i & 1][j], b[n][j], t, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][n][e] = __builtin_fmaf(f[n][g], t[e], acc[i][n][e]);
                }
        }
    };
    // Whole rounds of the ring have no branches, so that every wait in them is for the step's own loads only.
    const int whole = min(steps, a.K / (128 * KS));  // the end of the steps without a part past K
    int c0 = first;
    for (; c0 + PF <= whole; c0 += PF)
        [&]<int... U>(std::integer_sequence<int, U...>) {
            (step(std::integral_constant<int, U>{}, c0 + U, true), ...);
        }(std::make_integer_sequence<int, PF>{});
    for (; c0 < steps; c0 += PF)
        [&]<int... U>(std::integer_sequence<int, U...>) {
            ((c0 + U < steps && (step(std::integral_constant<int, U>{}, c0 + U, false), true)) && ...);
        }(std::make_integer_sequence<int, PF>{});
    // the accesses behind the last step are done with the stages too
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(qt_vmcnt(0));
    hx_lds_barrier();
    if constexpr (KS > 1) {  // the parts' sums, in order; part p finishes row blocks p, p + KS, ..
        static_assert(NT <= PF, "the sums fit the stages");
        hx_f4* red = reinterpret_cast<hx_f4*>(w4_lds);  // [KS][4][RB][NT][64]
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) red[((wave * RB + i) * NT + n) * 64 + lane] = acc[i][n];
        hx_lds_barrier();
#pragma unroll
        for (int i = 0; i < RB; ++i)
            if (i % KS == part)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    hx_f4 v = red[((cw * RB + i) * NT + n) * 64 + lane];
#pragma unroll
                    for (int p = 1; p < KS; ++p) v += red[(((4 * p + cw) * RB + i) * NT + n) * 64 + lane];
                    acc[i][n] = v;
                }
    }
    if (sp.splits > 1) {  // the splits' sums, in order: the last workgroup of a tile to arrive adds them
        constexpr int PIECES = RB * NT * 256;
        hx_f4* mine = sp.partial + (size_t)tile * sp.splits * PIECES;
        const __amdgpu_buffer_rsrc_t rp = coherent_rsrc(mine);
#pragma unroll
        for (int i = 0; i < RB; ++i)
            if (i % KS == part)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    coherent_store4(rp, (split * PIECES + ((i * NT + n) * 4 + cw) * 64 + lane) * 16, acc[i][n]);
        if (!arrive_last(sp.counters + tile, sp.splits)) return;
#pragma unroll
        for (int i = 0; i < RB; ++i)
            if (i % KS == part)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int at = (((i * NT + n) * 4 + cw) * 64 + lane) * 16;
                    hx_f4 v = coherent_load4(rp, at);
                    for (int p = 1; p < sp.splits; ++p) v += coherent_load4(rp, at + p * PIECES * 16);
                    acc[i][n] = v;
                }
    }
#pragma unroll
    for (int i = 0; i < RB; ++i)
        if (i % KS == part)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int nn = n0 + 16 * (cw * NT + n) + col;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int m = m0 + 16 * i + 4 * kg + e;
                    if (m < M && nn < a.N) store_y(y, (size_t)m * a.N + nn, acc[i][n][e], y_fp32);
                }
            }
}

template <int BM, int NT, int KS, int PF, int GS, bool Z, bool V>
__global__ __launch_bounds__(256 * KS) void w4_tile_kernel(const _Float16* x, W4Args a, void* y, int M, bool y_fp32, W4Split sp)
{
    w4_tile<BM, NT, KS, PF, GS, Z, V>(x, a, y, M, y_fp32, sp);
}

// out[t][k] = scale * weight(tokens[t], k), rounded once to fp32 (and once more where T is fp16); zeros for a token outside [0, N).
// One thread per word: 8 consecutive outputs.  total: words, below 2^31, so that a division of 32 bits finds the row.  Memory
// bound: 20000 rows of 4096 43 us, 4.8 TB/s; 2000 6.5 us, of which launch and latency are 2.5.
template <typename T>
__global__ __launch_bounds__(256) void w4_embed_kernel(W4Args a, const int64_t* tokens, T* out, uint32_t total, float scale)
{
    typedef T v8 __attribute__((ext_vector_type(8)));
    const uint32_t nw = (uint32_t)(a.K + 127) / 128 * 16, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const uint32_t t = i / nw, w = i % nw;
    const int k = word_k((int)w);
    if (k >= a.K) return;
    const int64_t row = tokens[t];
    v8 o = {};
    if (row >= 0 && row < a.N) {
        const size_t g = (size_t)row * a.groups + (k >> a.group_log2);
        float v[8];
        word_values(a.words[(size_t)row * nw + w], a.zeros ? (float)a.zeros[g] : 8.0f, v);
        const float s = (float)a.scales[g];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (T)(v[j] * s * scale);  // v * s is exact: 9 bits times 11
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
    void* ws;  // counters and the splits' sums, or null
    hipStream_t st;
};

// Which kernel takes a call of M rows, by measured shapes (us, 4-bit, group 128, weights from memory).
struct W4Plan {
    enum Kind { ROWS4_FEW, ROWS4, ROWS8_FEW, ROWS8, ROWS8_WIDE, TILE16, TILE32, TILE64, TILE64W, TILE64W2, TILE128 } kind;
    int splits, steps;  // of a tile kernel
    long tiles;
};
struct W4Tile {
    int bm, nt, ks;
};
constexpr W4Tile W4_TILES[] = {{16, 1, 2}, {32, 1, 2}, {64, 1, 2}, {64, 2, 1}, {64, 2, 2}, {128, 2, 1}};  // TILE16 ..
constexpr int W4_SLOTS = 256;  // workgroups that splitting fills the chip with, one per CU

W4Plan w4_tile_plan(int kind, int M, int N, int K, int splits)
{
    const W4Tile t = W4_TILES[kind - W4Plan::TILE16];
    const int steps = (K + 128 * t.ks - 1) / (128 * t.ks);
    W4Plan p{(W4Plan::Kind)kind, 1, (steps + splits - 1) / splits, 0};
    p.splits = (steps + p.steps - 1) / p.steps;
    p.tiles = ((long)M + t.bm - 1) / t.bm * (((long)N + 64 * t.nt - 1) / (64 * t.nt));
    return p;
}

// gs: groups in a block of 128 k.  pieces: the kernels for groups in aligned pieces are among the choice; the others are built for the
// basic shapes only.  Measured as groups of 128 without zero points / of 32 with.
W4Plan w4_plan(int M, int N, int K, int gs, bool split, bool pieces)
{
    // Few weights: 2 loads per wave, so that more waves share them (1 row, 4096 -> 2048: 3.9 / 4.4 us, 4.4 / 4.9 with 4 loads; 8192 ->
    // 4096 7.3 / 8.7 and 7.4 / 8.3, with 4 rows 10.6 / 11.5 and 8.6 / 9.5).  Of many, the groups of 32 take the place that
    // more loads need (1 row, 4096 -> 12288 9.7 / 11.3 and 9.1 / 12.5; -> 32768 20.4 / 23.6 and 18.6 / 25.9).
    if (M <= 4) return {!pieces || N < 4096 || (gs == 4 && N > 8192) ? W4Plan::ROWS4_FEW : W4Plan::ROWS4, 1, 0, 0};
    // 5 rows as 16 waves of one load / 8 waves of 2 / 8 waves of 2 in each of two spans: 4096 -> 2048 4.9, 5.8, 6.0 us (groups of 32
    // 5.1, 6.2, 6.7); 2048 -> 2048 4.7, 4.2, 5.8; 8192 -> 4096 13.5, 8.5, 9.9; 2048 -> 8192 8.1, 5.6, 6.1; 4096 -> 12288
    // 15.5, 11.4, 10.5 (17.3, 12.4, 15.5); -> 32768 33, 25, 20.5 (38, 27.6, 29.6).
    if (M <= 8) {
        const W4Plan::Kind kind = N < 4096 && K >= 4096 ? W4Plan::ROWS8_FEW : N > 8192 && gs < 4 ? W4Plan::ROWS8_WIDE : W4Plan::ROWS8;
        return {pieces ? kind : W4Plan::ROWS8, 1, 0, 0};
    }
    // A step of a tile, in us, where there is at most one workgroup for two CUs, where there is one per CU, and per workgroup where
    // there are more; how much longer groups of 32 with zero points take.  K is split among workgroups of the tiles with one
    // column group per wave where CUs are idle.  64 rows, 64-row tiles: 16384 -> 4096 41 us unsplit, 21.5 in 4; 8192 -> 4096 25 and 14.7.
    // 64 rows of 2048 -> 8192 9.1 us in tiles of 64, 7.8 of 32; 128 rows of 4096 -> 12288 32 us in tiles of 64, 28 and 24 in the two of 64 x
    // 128, 34 of 128; 256 rows of 4096 -> 32768 122, 83, 93 and 70 us.
    struct Cost {
        int kind;
        float few, one, more, fine;
    };
    constexpr Cost cost[] = {{W4Plan::TILE16, 0.35f, 0.45f, 0.51f, 1.25f}, {W4Plan::TILE32, 0.43f, 0.56f, 0.62f, 1.25f},
                             {W4Plan::TILE64, 0.68f, 0.86f, 0.92f, 1.2f},  {W4Plan::TILE64W, 0.56f, 0.77f, 0.62f, 1.4f},
                             {W4Plan::TILE64W2, 1.15f, 1.32f, 1.4f, 1.42f}, {W4Plan::TILE128, 0.96f, 1.36f, 1.03f, 1.25f}};
    W4Plan best{};
    float least = 1e30f;
    for (const Cost& c : cost) {
        const W4Tile t = W4_TILES[c.kind - W4Plan::TILE16];
        if ((c.kind == W4Plan::TILE16 ? M > 16 : M <= t.bm / 2) || (t.nt > 1 && !pieces)) continue;
        for (int splits = 1; splits <= (split && t.nt == 1 ? 8 : 1); splits *= 2) {
            const W4Plan p = w4_tile_plan(c.kind, M, N, K, splits);
            const long n = p.tiles * p.splits;
            if (splits > 1 && (n > W4_SLOTS || p.steps < 2)) break;
            const float step = n <= W4_SLOTS / 2 ? c.few : n <= W4_SLOTS ? c.one : (float)((n + W4_SLOTS - 1) / W4_SLOTS) * c.more;
            const float join = splits > 1 ? 0.6f + (float)splits * (0.55f + 0.005f * (float)t.bm) : 0.0f;
            const float us = (float)p.steps * step * (gs == 4 ? c.fine : gs == 2 ? 0.5f + 0.5f * c.fine : 1.0f) + join;
            if (us < least) least = us, best = p;
        }
    }
    return best;
}

size_t w4_partial_bytes(const W4Plan& p)
{
    const W4Tile t = W4_TILES[p.kind - W4Plan::TILE16];
    return (size_t)p.tiles * p.splits * t.bm * 64 * t.nt * sizeof(float);
}

template <int S, int WAVES, int NS, int NT, int GS, bool Z, bool V>
hipError_t rows_launch(const W4Call& c)
{
    const int spans = ((c.a.K + 127) / 128 + S - 1) / S;
    int wk = 1;  // waves along K: as many as have spans, up to all
    while (wk < WAVES && wk * NS < spans) wk *= 2;
    const int rows = WAVES / wk * NT * 16 / S, tiles = (c.a.N + rows - 1) / rows;
    hipLaunchKernelGGL((w4_rows_kernel<S, WAVES, NS, NT, GS, Z, V>), dim3(tiles < 2 * W4_SLOTS ? tiles : 2 * W4_SLOTS), dim3(64 * WAVES), 0, c.st, c.x, c.a, c.y,
                       c.M, c.y_fp32, wk);
    return hipGetLastError();
}

template <int BM, int NT, int KS, int PF, int GS, bool Z, bool V>
hipError_t tile_launch(const W4Call& c, const W4Plan& p)
{
    constexpr size_t lds = sizeof(_Float16) * PF * KS * BM * 128;
    const W4Split sp{p.splits, p.steps, reinterpret_cast<hx_f4*>(static_cast<char*>(c.ws) + HX_COUNTER_BYTES),
                     static_cast<int*>(c.ws)};
    hipLaunchKernelGGL((w4_tile_kernel<BM, NT, KS, PF, GS, Z, V>), dim3((unsigned)(p.tiles * p.splits)), dim3(256 * KS), lds,
                       c.st, c.x, c.a, c.y, c.M, c.y_fp32, sp);
    return hipGetLastError();
}

template <int GS, bool Z, bool V>
hipError_t gemm_launch(const W4Call& c)
{
    const W4Plan p = w4_plan(c.M, c.a.N, c.a.K, GS, c.ws != nullptr, V || GS == 1);
    if constexpr (V || GS == 1) {
        switch (p.kind) {
            case W4Plan::ROWS4: return rows_launch<4, 8, 1, 4, GS, Z, V>(c);
            case W4Plan::ROWS8_FEW: return rows_launch<2, 16, 1, 1, GS, Z, V>(c);
            case W4Plan::ROWS8_WIDE: return rows_launch<2, 8, 2, 2, GS, Z, V>(c);
            case W4Plan::TILE64W: return tile_launch<64, 2, 1, 4, GS, Z, V>(c, p);
            case W4Plan::TILE64W2: return tile_launch<64, 2, 2, 4, GS, Z, V>(c, p);
            case W4Plan::TILE128: return tile_launch<128, 2, 1, 2, GS, Z, V>(c, p);
            default: break;
        }
    }
    switch (p.kind) {
        case W4Plan::ROWS4_FEW: return rows_launch<4, 8, 1, 2, GS, Z, V>(c);
        case W4Plan::ROWS8: return rows_launch<2, 8, 1, 2, GS, Z, V>(c);
        case W4Plan::TILE16: return tile_launch<16, 1, 2, 4, GS, Z, V>(c, p);
        case W4Plan::TILE32: return tile_launch<32, 1, 2, 4, GS, Z, V>(c, p);
        default: return tile_launch<64, 1, 2, 4, GS, Z, V>(c, p);
    }
}

template <int GS, bool Z>
hipError_t gemm_launch(const W4Call& c)
{
    if constexpr (GS == 1) {
        return gemm_launch<GS, Z, true>(c);
    } else {
        const bool pieces = c.a.groups % GS == 0 && reinterpret_cast<uintptr_t>(c.a.scales) % (2 * GS) == 0 &&
                            reinterpret_cast<uintptr_t>(c.a.zeros) % GS == 0;
        return pieces ? gemm_launch<GS, Z, true>(c) : gemm_launch<GS, Z, false>(c);
    }
}

template <int GS>
hipError_t gemm_launch(const W4Call& c)
{
    return c.a.zeros ? gemm_launch<GS, true>(c) : gemm_launch<GS, false>(c);
}

}  // namespace

// Bytes of workspace with which calls of M rows split K; 0 where none do.  Splits come in W4_SLOTS workgroups of 64 x 64 sums at most:
// 4 MiB and the counters.
size_t w4_gemm_workspace_bytes(int M, int N, int K)
{
    size_t most = 0;
    for (const int gs : {1, 2, 4})
        for (const bool pieces : {false, true}) {
            const W4Plan p = w4_plan(M, N, K, gs, true, pieces);
            if (p.splits > 1 && w4_partial_bytes(p) > most) most = w4_partial_bytes(p);
        }
    return most ? HX_COUNTER_BYTES + most : 0;
}

hipError_t launch_w4_gemm(const _Float16* x, const W4Args& a, void* y, int M, bool y_fp32, void* ws, size_t ws_bytes,
                          hipStream_t st)
{
    // 2^20 tiles of 64 x 64 and fewer in a launch: one takes at most 2^32 threads
    const long columns = ((long)a.N + 63) / 64, most = 64 * (columns < 1l << 20 ? (1l << 20) / columns : 1);
    for (long m = 0; m < M; m += most) {
        const int rows = (int)(M - m < most ? M - m : most);
        const size_t need = w4_gemm_workspace_bytes(rows, a.N, a.K);
        const W4Call c{x + m * a.K, a, static_cast<char*>(y) + m * a.N * (y_fp32 ? 4 : 2), rows, y_fp32,
                       need && ws && ws_bytes >= need ? ws : nullptr, st};
        const hipError_t e = a.group_log2 == 5 ? gemm_launch<4>(c) : a.group_log2 == 6 ? gemm_launch<2>(c) : gemm_launch<1>(c);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_w4_embed(const W4Args& a, const int64_t* tokens, void* out, int n, float scale, bool out_fp32,
                           hipStream_t st)
{
    if (n <= 0) return hipSuccess;
    const int nw = (a.K + 127) / 128 * 16, most = (int)((1u << 31) / nw) - 1;  // rows of a launch
    for (int t = 0; t < n; t += most) {
        const uint32_t total = (uint32_t)(n - t < most ? n - t : most) * nw;
        const dim3 grid((total + 255) / 256);
        if (out_fp32)
            hipLaunchKernelGGL((w4_embed_kernel<float>), grid, dim3(256), 0, st, a, tokens + t,
                               static_cast<float*>(out) + (size_t)t * a.K, total, scale);
        else
            hipLaunchKernelGGL((w4_embed_kernel<_Float16>), grid, dim3(256), 0, st, a, tokens + t,
                               static_cast<_Float16*>(out) + (size_t)t * a.K, total, scale);
        if (n - t <= most) break;
    }
    return hipGetLastError();
}

}  // namespace hx
