// hx_beam.hip -- one step of beam search on gfx950: the best continuations over beams and vocabulary, and the surviving
// beams' states.
//
//   score(w, v) = cum[w] + (logit[w][v] - logsumexp_v logit[w]),  the n best of each sequence in descending order,
//   the lowest w * vocab + v first among equals
//
// A finished beam (done[w] != 0) has one candidate, (w, eos) with score cum[w].  A beam whose cum is not finite, whose logits
// hold a NaN or +inf, or are all -inf, has none (its log-softmax is not defined); a logit of -inf is no candidate.
// Sequences with fewer than n candidates get score -inf, parent -1 and token -1 behind them.
//
// Selection is one launch.  A workgroup takes one chunk of one row and reads it once, in pieces of 4096 logits with the next
// two in flight: running maximum and sum of exponentials per thread, and which blocks (the 16 logits of a thread and piece) may
// hold some of the n largest.  Few blocks are left at the end; their logits are read again and ranked.  The last workgroup of
// a sequence to arrive merges the chunks: the rows' log-sum-exp and the candidates' scores from their sums in 64 bits, the n best.
//
// Error of a log-sum-exp, with p pieces in a chunk: 1e-6 from the exponentials' fp32 arguments (2^-24 + 2^-26 of x - max, whose mean under
// the softmax is at most ln vocab), 15 + p additions of a thread, 9 of a workgroup, p + 1 rescalings of 2^-22 at most, two roundings of the
// reference: 4e-6 + 3e-7 p.  It does not depend on the logits' size.
//
// The n largest of a set spread over threads, without sorting it: the n-th largest of the threads' maxima is a lower bound of
// the n-th largest of all, and only what reaches it (n to 2n of random elements) is ranked.  The bound is renewed after 1, 2,
// 4, .. pieces.
//
// 4 rows of 151552 fp32 logits, n = 8: 12.3 us, a chain of latencies beside 0.5 us of traffic: a piece's load 2.1, a bound and the ranking
// 1.8, the last arrival 1.9, then the merge 5.9 (sums of rows 2.3, candidates, bound and ranking 3.6).  256 rows in fp16, n = 16, a fifth of
// them finished and not read: 30 us, of which the last logits come at 18.4 (62 MB, 3.4 TB/s) and the last sequence's merge starts at 22.3.
#include "hx_gemv.hpp"
#include "hx_kernels.hpp"

namespace hx {

namespace {

typedef unsigned long long u64;

// Order-preserving key of a float that is no NaN (equal for -0 and +0): larger for larger values, never 0.
HX_INLINE uint32_t float_key(float x)
{
    const int u = __builtin_bit_cast(int, x + 0.0f);
    return (uint32_t)u ^ (uint32_t)((u >> 31) | (int)0x80000000);
}
HX_INLINE float key_float(uint32_t k) { return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;

// i / d for i < 2^32, with m = ceil(2^32 / d): the product's high word is the quotient or one more.
struct FastDiv {
    uint32_t d, m;
};
HX_INLINE uint32_t div_by(uint32_t i, FastDiv f)
{
    if (f.d == 1) return i;
    const uint32_t q = __umulhi(i, f.m);
    return q * (u64)f.d > i ? q - 1 : q;
}

// A lower bound of the n-th largest of 64 P keys in LDS, for one wave (0 where fewer than n are above 0): the key's 20 high bits from the
// top, two at a time, each pair as large as still leaves n keys at or above the value, then the least of the keys that reach it (equal
// keys give their own value).  Keys above 0 are no less than KEY_NEG_INF.
template <int P>
HX_INLINE uint32_t nth_largest(const uint32_t* keys, int n)
{
    const int lane = threadIdx.x & 63;
    uint32_t k[P];
#pragma unroll
    for (int p = 0; p < P; ++p) k[p] = keys[64 * p + lane];
    uint32_t t = 0;
    for (int bit = 30; bit >= 12; bit -= 2) {
        int count[4] = {};
#pragma unroll
        for (int d = 1; d < 4; ++d)
#pragma unroll
            for (int p = 0; p < P; ++p) count[d] += __popcll(__ballot(k[p] >= (t | (uint32_t)d << bit)));
        t |= (uint32_t)(count[3] >= n ? 3 : count[2] >= n ? 2 : count[1] >= n ? 1 : 0) << bit;
    }
    uint32_t most = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) most = max(most, k[p] >= t ? ~k[p] : 0u);
    return t ? ~hx_wave_max_u32(most) : 0u;
}

// Lower bound of the n-th largest of all elements from the threads' largest keys (0: none): the n-th largest of the 256, or for
// small n of the 64 maxima of 4 adjacent threads, which is a third of the steps and a slightly lower bound.
HX_INLINE uint32_t bound_of(uint32_t key, int n, uint32_t* keys)
{
    __shared__ uint32_t bound;
    if (n <= 32) {
        key = max(key, (uint32_t)__shfl_xor((int)key, 1, 64));
        key = max(key, (uint32_t)__shfl_xor((int)key, 2, 64));
        if ((threadIdx.x & 3) == 0) keys[threadIdx.x >> 2] = key;
    } else {
        keys[threadIdx.x] = key;
    }
    hx_lds_barrier();
    if (hx_vwave() == 0) {  // another SIMD for each of the workgroups that share a CU
        const uint32_t t = n <= 32 ? nth_largest<1>(keys, n) : nth_largest<4>(keys, n);
        if ((threadIdx.x & 63) == 0) bound = t;
    }
    hx_lds_barrier();
    return bound;
}

// Over the 64 lanes, with lane-permuted operands instead of round trips through the LDS crossbar; every lane gets the result.
HX_INLINE float wave_max(float v) { return key_float(hx_wave_max_u32(float_key(v))); }
HX_INLINE float wave_sum(float v)
{
    auto add = [&](auto ctrl, auto rows) {
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value,
                                                                   decltype(rows)::value, 0xf, false));
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // row_shr:1
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});  // row_shr:2
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});  // row_shr:4
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});  // row_shr:8
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast:31
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Over groups of g lanes (a power of two), every lane gets the result: partners by lane permutations up to 16 lanes, then rows swapped.
template <typename T, typename F>
HX_INLINE T group_reduce(T v, int g, F f)
{
    struct Words {
        uint32_t w[sizeof(T) / 4];
    };
    auto with = [&](auto ctrl) {
        Words a = __builtin_bit_cast(Words, v);
#pragma unroll
        for (uint32_t& x : a.w) x = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(ctrl)::value, 0xf, 0xf, true);
        v = f(v, __builtin_bit_cast(T, a));
    };
    auto swapped = [&](auto half) {  // 32 lanes or rows of 16: the two results are the two sides, in all lanes
        Words a = __builtin_bit_cast(Words, v), b;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 4); ++i) {
            const auto r = decltype(half)::value ? __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false)
                                                 : __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
            a.w[i] = r[0], b.w[i] = r[1];
        }
        v = f(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
    };
    if (g > 1) with(std::integral_constant<int, 0xb1>{});   // quad_perm 1 0 3 2
    if (g > 2) with(std::integral_constant<int, 0x4e>{});   // quad_perm 2 3 0 1
    if (g > 4) with(std::integral_constant<int, 0x141>{});  // row_half_mirror
    if (g > 8) with(std::integral_constant<int, 0x140>{});  // row_mirror
    if (g > 16) swapped(std::integral_constant<int, 0>{});
    if (g > 32) swapped(std::integral_constant<int, 1>{});
    return v;
}

struct BeamPlan {
    int subs, chunks, lists;   // pieces of 4096 logits in a chunk; chunks of a row; beams * chunks, the lists of a sequence
    FastDiv by_chunks, by_lists;
    int cap;                   // candidates (16 bytes) that the merge's LDS buffer holds
    u64* entries;              // [batch][n][lists]: the r-th best of each list, key << 32 | ~token, 0: none
    float2* stats;             // [batch][lists]: the chunk's maximum, the sum of exp(logit - maximum)
    int* counters;             // arrivals per sequence
};

constexpr int SEL_THREADS = 256;
constexpr int SEL_E = 16;                           // logits of a thread in a piece
constexpr int PIECE = SEL_THREADS * SEL_E;
constexpr int BLOCKS = 4 * SEL_THREADS;              // entries of a chunk's list of blocks
constexpr int MERGE_E = 8;                          // candidates of a thread in one round of the merge
constexpr int MERGE = SEL_THREADS * MERGE_E;        // and of the workgroup

// A candidate of the merge: its score (-inf: none) and beam << 32 | token, in whose order equal scores come.
struct Cand {
    double s;
    u64 at;
};
HX_INLINE bool better(double s, u64 at, double s2, u64 at2) { return s > s2 || (s == s2 && at < at2); }

HX_INLINE u64 coherent_load8(__amdgpu_buffer_rsrc_t r, int off)
{
    return __builtin_bit_cast(u64, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, HX_BUF_SC1));
}
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
HX_INLINE void coherent_store8(__amdgpu_buffer_rsrc_t r, int off, u64 v)
{
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2v, v), r, off, 0, HX_BUF_SC1);
}

// Sums of exponentials are relative to 2^ref(top), top log2 e in fp32, or where that overflows (a maximum beyond REF_MAX) relative
// to e^top.  ref_rest(top) is what the rounding of ref left out: relative to e^top the former are 2^-ref_rest times as much.
// A maximum of +inf or a NaN makes the sum a NaN.  log2 e itself rounded to fp32 is off by 1.3e-8, which changes a
// log-sum-exp by that times the row's entropy, at most 2e-7.
constexpr float LOG2E = 1.44269504f, REF_MAX = 2e38f;
HX_INLINE bool ref_fits(float top) { return fabsf(top) < REF_MAX; }
HX_INLINE float ref_rest(float top) { return ref_fits(top) ? __builtin_fmaf(top, LOG2E, -(top * LOG2E)) : 0.0f; }
// Factor that takes a sum relative to `from` to one relative to the larger `to`.  The references are the rounded products: one fused
// into the subtraction would leave its rounding in the sum, up to 5e-6 of it for logits near 100 and 2.7e-3 near 60000.
HX_INLINE float rescale(float from, float to)
{
#pragma clang fp contract(off)
    return __builtin_amdgcn_exp2f(ref_fits(from) && ref_fits(to) ? from * LOG2E - to * LOG2E : (from - to) * LOG2E);
}

// SEL_E logits of a thread: element i is logit (i / VEC * SEL_THREADS + t) * VEC + i % VEC of its piece.
template <typename T>
struct Piece {
    static constexpr int VEC = 16 / sizeof(T), NV = SEL_E / VEC;
    typedef T vec __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
    vec v[NV];
    static HX_INLINE int offset(int t, int i) { return (i / VEC * SEL_THREADS + t) * VEC + i % VEC; }
    HX_INLINE void load(const T* x)
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = *reinterpret_cast<const vec*>(x + offset(threadIdx.x, i * VEC));
    }
    // Thread t's share of a piece of which only `room` logits are there; what lies behind is -inf.
    HX_INLINE void load_end(const T* x, int t, int room)
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int o = offset(t, i * VEC);
            if (o + VEC <= room) {
                v[i] = *reinterpret_cast<const vec*>(x + o);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[i][j] = o + j < room ? x[o + j] : (T)-INFINITY;
            }
        }
    }
    HX_INLINE float operator[](int i) const { return (float)v[i / VEC][i % VEC]; }
    HX_INLINE float most() const
    {
        vec t = v[0];
#pragma unroll
        for (int i = 1; i < NV; ++i) t = __builtin_elementwise_max(t, v[i]);
        float r = (float)t[0];
        if constexpr (sizeof(T) == 2) {  // two at a time down to the last pair
            hx_h4 h = __builtin_elementwise_max(hx_h4{t[0], t[1], t[2], t[3]}, hx_h4{t[4], t[5], t[6], t[7]});
            hx_h2 q = __builtin_elementwise_max(hx_h2{h[0], h[1]}, hx_h2{h[2], h[3]});
            r = fmaxf((float)q[0], (float)q[1]);
        } else {
#pragma unroll
            for (int j = 1; j < VEC; ++j) r = fmaxf(r, (float)t[j]);
        }
        return r;
    }
    // Sum of the exponentials relative to top (0 where that is -inf): one multiply-add and one exponential per logit.
    HX_INLINE float sum(float top) const
    {
        float s = 0.0f;
        if (ref_fits(top) || top == -INFINITY) {
            const float r = top == -INFINITY ? 0.0f : top * LOG2E;
#pragma unroll
            for (int i = 0; i < SEL_E; ++i) s += __builtin_amdgcn_exp2f(__builtin_fmaf((*this)[i], LOG2E, -r));
        } else {
#pragma unroll
            for (int i = 0; i < SEL_E; ++i) s += __builtin_amdgcn_exp2f(((*this)[i] - top) * LOG2E);
        }
        return s;
    }
};

HX_INLINE u64 wave_max_u64(u64 m)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const u64 q = __shfl_xor(m, o, 64);
        m = q > m ? q : m;
    }
    return m;
}

// Ranks the c candidates in LDS and puts the n best, in order, into `sorted`; returns how many there are.  The buffer is filled up
// with zeros to the next 16, which the loop takes at a time: one by one, each waited for the LDS (7 us for 184).  Starts and ends
// with a barrier.
HX_INLINE int rank_entries(u64* cand, int c, int n, u64* sorted)
{
    if ((int)threadIdx.x < (-c & 15)) cand[c + threadIdx.x] = 0;
    hx_lds_barrier();
    for (int i = threadIdx.x; i < c; i += SEL_THREADS) {
        const u64 mine = cand[i];
        int r = 0;
        for (int j = 0; j < c; j += 16) {
            ulonglong2 t[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) t[u] = reinterpret_cast<const ulonglong2*>(cand + j)[u];
#pragma unroll
            for (int u = 0; u < 8; ++u) r += (t[u].x > mine) + (t[u].y > mine);
        }
        if (r < n) sorted[r] = mine;
    }
    hx_lds_barrier();
    return min(c, n);
}

// Chunk `chunk` of a row, as list `list` of sequence b.
//
// Blocks are ordered by their maximum, then by their piece: logits of an earlier piece have lower tokens, so a block with n
// blocks before it in that order holds none of the n best.  (Blocks of one piece with equal maxima are not told apart.)
template <typename T>
HX_INLINE void select_chunk(const T* x, int chunk, int list, const BeamArgs& a, const BeamPlan& p, long b, char* lds)
{
    __shared__ uint32_t keys[SEL_THREADS];
    __shared__ u64 sorted[BEAM_MAX_N + SEL_THREADS];
    __shared__ u64 best[4];
    __shared__ float part[2][4];
    __shared__ int count;
    u64* cand = reinterpret_cast<u64*>(lds);  // [BLOCKS]: key of the maximum << 32 | ~(piece * SEL_THREADS + thread)
    const int tid = threadIdx.x, wave = tid >> 6, n = a.n;
    const int first = chunk * p.subs * PIECE, end = min(first + p.subs * PIECE, a.vocab);
    const int whole = (end - first) / PIECE;  // pieces; what is left over ends the row
    const bool over = first + whole * PIECE < end;
    float m = -INFINITY, sum = 0.0f;  // of this thread: its maximum; its exponentials, relative to that
    uint32_t need = 1, bound = 0;     // keys: what a block has to reach, what n logits reach
    int free = 0;                     // pieces that the list has room for in any case
    if (tid == 0) count = 0;
    auto take = [&](const Piece<T>& piece, int s) {
        const float most = piece.most();  // a NaN is skipped here and makes the sum a NaN below
        const float top = fmaxf(m, most);
        sum = (m == top ? sum : sum * rescale(m, top)) + piece.sum(top);
        m = top;
        // The threads' maxima so far give a bound that n blocks reach: from then on equals come too late.
        uint32_t now = need;
        if ((s & (s + 1)) == 0) {
            bound = max(bound, bound_of(float_key(m), n, keys));  // its barriers publish count
            now = max(need, bound), need = bound + 1;
        }
        if (free == 0) {
            int c = 0;
            if (s > 0) {
                hx_lds_barrier();
                c = count;
                hx_lds_barrier();  // every thread has read count
                if (c > BLOCKS - SEL_THREADS) {
                    c = rank_entries(cand, c, n + SEL_THREADS - 1, sorted);
                    for (int i = tid; i < c; i += SEL_THREADS) cand[i] = sorted[i];
                    if (tid == 0) count = c;
                    hx_lds_barrier();
                }
            }
            free = (BLOCKS - c) / SEL_THREADS;
        }
        --free;
        const uint32_t key = float_key(most);
        if (key >= now && most > -INFINITY)
            cand[atomicAdd(&count, 1)] = (u64)key << 32 | (uint32_t)~(uint32_t)(s * SEL_THREADS + tid);
    };
    Piece<T> block[2];  // the blocks that may hold some of the n largest, two per thread at most
    int base[2] = {first, first}, own[2] = {tid, tid};
    bool two = false;
    if (end - first <= PIECE) {
        if (over) block[0].load_end(x + first, tid, end - first);
        else block[0].load(x + first);
        take(block[0], 0);  // every thread keeps its block
    } else {
        // Two pieces in flight.  Every step loads one (past the end the last again), so that the waits are for the piece's own
        // loads.
        Piece<T> odd;
        block[0].load(x + first);
        odd.load(x + first + min(1, whole - 1) * PIECE);
        for (int s = 0; s < whole; s += 2) {
            take(block[0], s);
            block[0].load(x + first + min(s + 2, whole - 1) * PIECE);
            if (s + 1 < whole) take(odd, s + 1);
            odd.load(x + first + min(s + 3, whole - 1) * PIECE);
        }
        if (over) {
            block[0].load_end(x + first + whole * PIECE, tid, end - first - whole * PIECE);
            take(block[0], whole);
        }
        hx_lds_barrier();
        int c = count;
        hx_lds_barrier();
        if (c > SEL_THREADS) {
            // more than one per thread: those that reach the bound of all, or where they are many, the n + 255 first in order
            bound = max(bound, bound_of(float_key(m), n, keys));
            u64 mine[BLOCKS / SEL_THREADS];
#pragma unroll
            for (int i = 0; i < BLOCKS / SEL_THREADS; ++i) {
                const int at = i * SEL_THREADS + tid;
                mine[i] = at < c && (uint32_t)(cand[at] >> 32) >= bound ? cand[at] : 0;
            }
            if (tid == 0) count = 0;
            hx_lds_barrier();  // the list is read
#pragma unroll
            for (int i = 0; i < BLOCKS / SEL_THREADS; ++i)
                if (mine[i]) cand[atomicAdd(&count, 1)] = mine[i];
            hx_lds_barrier();
            c = count;
            hx_lds_barrier();
            if (c > 2 * SEL_THREADS) {
                c = rank_entries(cand, c, n + SEL_THREADS - 1, sorted);  // < 2 SEL_THREADS
                for (int i = tid; i < c; i += SEL_THREADS) cand[i] = sorted[i];
                hx_lds_barrier();
            }
            two = c > SEL_THREADS;
        }
        // their logits again
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (k == 0 || two) {
                const int at = k * SEL_THREADS + tid;
                const uint32_t id = at < c ? (uint32_t)~(uint32_t)cand[at] : 0;
                own[k] = id % SEL_THREADS;
                base[k] = first + (int)(id / SEL_THREADS) * PIECE;
                block[k].load_end(x + base[k], own[k], at < c ? end - base[k] : 0);
            }
    }
    const float wm = wave_max(m);
    if ((tid & 63) == 0) part[0][wave] = wm;
    hx_lds_barrier();  // the list is read
    if (tid == 0) count = 0;
    hx_lds_barrier();
    const float least = bound > KEY_NEG_INF ? key_float(bound) : -3.402823466e38f;
    auto entry = [&](int k, int i) {
        const int token = base[k] + Piece<T>::offset(own[k], i);
        return (u64)float_key(block[k][i]) << 32 | (uint32_t)~(uint32_t)token;
    };
    auto reach = [&](int k) {
#pragma unroll
        for (int i = 0; i < SEL_E; ++i)
            if (block[k][i] >= least) {
                const int at = atomicAdd(&count, 1);
                if (at < BLOCKS) cand[at] = entry(k, i);
            }
    };
    reach(0);
    if (two) reach(1);
    hx_lds_barrier();
    int found = count;
    if (found <= BLOCKS) {
        found = rank_entries(cand, found, n, sorted);
    } else {  // ties at the bound: one after the other
        u64 last = ~0ull;
        for (int r = 0; r < n; ++r) {
            u64 q = 0;
            auto next = [&](int k) {
#pragma unroll
                for (int i = 0; i < SEL_E; ++i) {
                    const u64 e = block[k][i] >= least ? entry(k, i) : 0;
                    if (e < last && e > q) q = e;
                }
            };
            next(0);
            if (two) next(1);
            q = wave_max_u64(q);
            if ((tid & 63) == 0) best[wave] = q;
            hx_lds_barrier();
            const u64 h = best[0] > best[1] ? best[0] : best[1], g = best[2] > best[3] ? best[2] : best[3];
            last = h > g ? h : g;
            if (tid == 0) sorted[r] = last;
            hx_lds_barrier();  // best is read before the next round's
        }
        found = n;  // more than n reach the bound
    }
    const float top = fmaxf(fmaxf(part[0][0], part[0][1]), fmaxf(part[0][2], part[0][3]));
    // a thread without finite logits has m = -inf and a sum of 0 (or a NaN)
    sum = wave_sum((m == top ? sum : sum * rescale(m, top)) * __builtin_amdgcn_exp2f(-ref_rest(top)));
    if ((tid & 63) == 0) part[1][wave] = sum;
    const __amdgpu_buffer_rsrc_t out = coherent_rsrc(p.entries + (size_t)b * a.n * p.lists + list);
    for (int r = tid; r < n; r += SEL_THREADS) coherent_store8(out, r * p.lists * 8, r < found ? sorted[r] : 0);
    hx_lds_barrier();
    if (tid == 0) {
        const float2 st = {top, (part[1][0] + part[1][1]) + (part[1][2] + part[1][3])};
        coherent_store8(coherent_rsrc(p.stats + (size_t)b * p.lists + list), 0, __builtin_bit_cast(u64, st));
    }
}

// The n best of the sequence's candidates.  lds: offset [beams] double, top [beams] float, then the candidate buffer.
HX_INLINE void select_merge(const BeamArgs& a, const BeamPlan& p, long b, char* lds)
{
    __shared__ uint32_t keys[SEL_THREADS];
    __shared__ Cand carry[BEAM_MAX_N];  // the best so far
    __shared__ Cand best[4];
    __shared__ int count, wanted[2][4];  // wanted: by round and wave
    double* offset = reinterpret_cast<double*>(lds);
    float* tops = reinterpret_cast<float*>(offset + a.beams);  // NaN: the beam is finished
    Cand* cand = reinterpret_cast<Cand*>(lds + ((size_t)a.beams * 12 + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 63, n = a.n, total = n * p.lists;
    const __amdgpu_buffer_rsrc_t rs = coherent_rsrc(p.stats + (size_t)b * p.lists);
    const __amdgpu_buffer_rsrc_t re = coherent_rsrc(p.entries + (size_t)b * n * p.lists);
    // A round takes the same number of entries beside the best so far, so that the next one's are on their way in each; the first
    // round's come while the rows' sums are formed.
    u64 e[MERGE_E];
    auto load = [&](int at) {
        const int fresh = min(total - at, MERGE - n);
#pragma unroll
        for (int i = 0; i < MERGE_E; ++i) {
            const int q = i * SEL_THREADS + tid;
            e[i] = q < fresh ? coherent_load8(re, (at + q) * 8) : 0;
        }
    };
    load(0);
    // score = offset[w] + (logit - tops[w]); offset NaN: the row has no candidates.  g lanes per row, as many as take all rows at once
    // (16 rows of 37 chunks, 32 candidates: 3 us less than with 64 lanes a row); first the maxima, then the sums relative to the row's.
    int g = 1;
    while (g < 64 && g < p.chunks && 2 * g * a.beams <= SEL_THREADS) g *= 2;
    for (int w0 = 0; w0 < a.beams; w0 += SEL_THREADS / g) {
        const int w = w0 + tid / g;
        const bool mine = w < a.beams;
        const float cum = mine ? a.cum[b * a.beams + w] : NAN;
        const bool fin = mine && a.done && a.done[b * a.beams + w];
        // of finished and dead rows: whatever is there
        auto chunk = [&](int c) {
            float2 st = {-INFINITY, 0.0f};
            if (mine && c < p.chunks) st = __builtin_bit_cast(float2, coherent_load8(rs, (w * p.chunks + c) * 8));
            return st;
        };
        float2 st = chunk(tid % g);
        float m = st.x;
#pragma unroll 4
        for (int c = tid % g + g; c < p.chunks; c += g) m = fmaxf(m, chunk(c).x);
        const float top = group_reduce(m, g, [](float x, float y) { return fmaxf(x, y); });
        double s = 0.0;
        for (int c = tid % g; c < p.chunks; c += g) {
            const float2 next = chunk(c + g);
            double e = (double)st.y;  // of a chunk without finite logits 0, or a NaN
            if (st.x != top && st.x > -INFINITY) e *= exp((double)st.x - (double)top);
            s += e;
            st = next;
        }
        s = group_reduce(s, g, [](double x, double y) { return x + y; });
        if (mine && tid % g == 0) {
            double off = NAN;
            if (!(fabsf(cum) < INFINITY)) {
            } else if (fin) {
                off = (double)cum;
            } else if (fabsf(top) < INFINITY && s < INFINITY) {  // a NaN fails both tests
                off = (double)cum - log(s);
            }
            offset[w] = off, tops[w] = fin ? NAN : top;
        }
    }
    int kept = 0, nothing = 0;  // entries of carry; entries in a row that were no better than those
    hx_lds_barrier();
    for (int at = 0, round = 0; at < total; ++round) {
        const int fresh = min(total - at, MERGE - n);
        Cand v[MERGE_E];
        const Cand last_kept = kept == n ? carry[n - 1] : Cand{-INFINITY, ~0ull};
        double most = -INFINITY;
        bool any = false;  // an entry that would be among the n best so far
#pragma unroll
        for (int h = 0; h < MERGE_E; h += 2) {
            v[h] = v[h + 1] = {-INFINITY, 0};
            if (h * SEL_THREADS >= fresh) continue;
            // two at a time without branches, so that they do not wait for each other's reads
            double off[2];
            float top[2];
            uint32_t beam[2];
            bool head[2];  // the row's first entry, which stands for a finished beam's only candidate
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t f = at + min((h + u) * SEL_THREADS + tid, fresh - 1), rank = div_by(f, p.by_lists), list = f - rank * p.lists;
                beam[u] = div_by(list, p.by_chunks);
                head[u] = rank == 0 && list == beam[u] * p.chunks;
                off[u] = offset[beam[u]];
                top[u] = tops[beam[u]];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const u64 entry = e[h + u];
                const bool fin = top[u] != top[u];
                const bool is = (h + u) * SEL_THREADS + tid < fresh && off[u] == off[u] && (fin ? head[u] : entry != 0);
                const double score = off[u] + ((double)key_float((uint32_t)(entry >> 32)) - (double)top[u]);
                Cand& c = v[h + u];
                c.s = is ? fin ? off[u] : score : -INFINITY;
                c.at = (u64)beam[u] << 32 | (fin ? (uint32_t)a.eos : (uint32_t)~(uint32_t)entry);
                any |= is && better(c.s, c.at, last_kept.s, last_kept.at);
                most = fmax(most, c.s);
            }
        }
        if (kept)
#pragma unroll
            for (int i = 0; i < MERGE_E; ++i) {
                const int q = i * SEL_THREADS + tid - fresh;
                if (q >= 0 && q < kept) v[i] = carry[q], most = fmax(most, v[i].s);
            }
        at += fresh;
        if (at < total) load(at);
        // so few that ranking them all costs less than a bound (1.5 us)
        const bool few = total <= 128;
        const u64 ask = __ballot(any);
        if (lane == 0) wanted[round & 1][tid >> 6] = ask != 0;
        hx_lds_barrier();
        const int* asked = wanted[round & 1];
        if (!(asked[0] | asked[1] | asked[2] | asked[3])) {
            // Every list is in descending order and the r-th entries of all lists come before the r+1-st: once an entry of each
            // list in turn was no better, none behind them is.
            nothing += fresh;
            if (nothing >= p.lists) break;
            continue;
        }
        nothing = 0;
        if (tid == 0) count = 0;
        // scores rounded to fp32 keep their order (not strictly): the bound holds for the rounded ones
        if (few) hx_lds_barrier();  // count
        const uint32_t bound = few ? 0 : bound_of(most > -INFINITY ? float_key((float)most) : 0, n, keys);
        if (most > -INFINITY && float_key((float)most) >= bound) {
#pragma unroll
            for (int i = 0; i < MERGE_E; ++i)
                if (v[i].s > -INFINITY && float_key((float)v[i].s) >= bound) {
                    const int to = atomicAdd(&count, 1);
                    if (to < p.cap) cand[to] = v[i];
                }
        }
        hx_lds_barrier();
        const int c = count;
        if (c <= p.cap) {
            if (tid < (-c & 7)) cand[c + tid] = {-INFINITY, ~0ull};
            hx_lds_barrier();
            for (int i = tid; i < c; i += SEL_THREADS) {
                const Cand mine = cand[i];
                int r = 0;
                for (int j = 0; j < c; j += 8) {  // 8 at a time, as in rank_entries
                    Cand t[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) t[u] = cand[j + u];
#pragma unroll
                    for (int u = 0; u < 8; ++u) r += better(t[u].s, t[u].at, mine.s, mine.at);
                }
                if (r < n) carry[r] = mine;
            }
            kept = min(c, n);
            hx_lds_barrier();
        } else {
            Cand last = {INFINITY, 0};
            for (int r = 0; r < n; ++r) {  // c > n: there are n to take
                Cand m = {-INFINITY, ~0ull};
#pragma unroll
                for (int i = 0; i < MERGE_E; ++i)
                    if (better(last.s, last.at, v[i].s, v[i].at) && better(v[i].s, v[i].at, m.s, m.at)) m = v[i];
#pragma unroll
                for (int o = 32; o >= 1; o >>= 1) {
                    const double s = __shfl_xor(m.s, o, 64);
                    const u64 i = __shfl_xor(m.at, o, 64);
                    if (better(s, i, m.s, m.at)) m = {s, i};
                }
                if (lane == 0) best[tid >> 6] = m;
                hx_lds_barrier();
                last = best[0];
                for (int i = 1; i < 4; ++i)
                    if (better(best[i].s, best[i].at, last.s, last.at)) last = best[i];
                if (tid == 0) carry[r] = last;
                hx_lds_barrier();
            }
            kept = n;
        }
    }
    for (int r = tid; r < n; r += SEL_THREADS) {
        const bool found = r < kept;
        a.scores[b * n + r] = found ? (float)carry[r].s : -INFINITY;
        a.parents[b * n + r] = found ? (int64_t)(carry[r].at >> 32) : -1;
        a.tokens[b * n + r] = found ? (int64_t)(uint32_t)carry[r].at : -1;
    }
}

}  // namespace

// grid: [batch][beams][chunks]
template <typename T>
__global__ __launch_bounds__(SEL_THREADS, 4) void beam_select_kernel(const T* logits, BeamArgs a, BeamPlan p)
{
    extern __shared__ __align__(16) char beam_lds[];
    const uint32_t row = div_by(blockIdx.x, p.by_chunks), chunk = blockIdx.x - row * p.chunks;
    const uint32_t b = div_by(blockIdx.x, p.by_lists), list = blockIdx.x - b * p.lists;
    // rows that are finished or dead are not read
    if (!(a.done && a.done[row]) && fabsf(a.cum[row]) < INFINITY)
        select_chunk(logits + row * a.ld, chunk, list, a, p, b, beam_lds);
    if (!arrive_last(p.counters + b, p.lists)) return;
    select_merge(a, p, b, beam_lds);
}

namespace {

// A chunk is as many pieces as leave about 4 workgroups per CU, which is what their registers allow at once.
struct SelectLayout {
    long subs, chunks, lists;
    size_t entries, stats, total;  // bytes
    SelectLayout(int batch, int beams, int vocab, int n)
    {
        const long pieces = ((long)vocab + PIECE - 1) / PIECE, rows = (long)batch * beams;
        const long per_row = 1024 / rows > 1 ? 1024 / rows : 1;  // chunks
        subs = (pieces + per_row - 1) / per_row;
        chunks = (pieces + subs - 1) / subs;
        lists = beams * chunks;
        entries = (size_t)batch * n * lists * sizeof(u64);
        stats = (size_t)batch * lists * sizeof(float2);
        total = HX_COUNTER_BYTES + entries + stats;
    }
};

FastDiv fast_div(uint32_t d) { return {d, (uint32_t)(((1ull << 32) + d - 1) / d)}; }

}  // namespace

// 0 for extents beyond what one launch can take (grid and 32-bit offsets within a sequence's lists).
size_t beam_select_workspace_bytes(int batch, int beams, int vocab, int n)
{
    const SelectLayout l(batch, beams, vocab, n);
    if ((long)batch * l.lists >= 1l << 23 || (long)n * l.lists >= 1l << 27) return 0;
    return l.total;
}

hipError_t launch_beam_select(const void* logits, bool fp32, const BeamArgs& a, void* ws, hipStream_t st)
{
    if (a.batch <= 0) return hipSuccess;
    const SelectLayout l(a.batch, a.beams, a.vocab, a.n);
    char* base = static_cast<char*>(ws);
    // the merge's candidates, 16 times what is asked for and more for few: ties aside a bound is reached by n to 2n as a rule
    const int cap = a.n > 8 ? 16 * a.n : 128;
    const BeamPlan p{(int)l.subs, (int)l.chunks, (int)l.lists, fast_div(l.chunks), fast_div(l.lists), cap,
                     reinterpret_cast<u64*>(base + HX_COUNTER_BYTES),
                     reinterpret_cast<float2*>(base + HX_COUNTER_BYTES + l.entries), reinterpret_cast<int*>(base)};
    const size_t merge = ((size_t)a.beams * 12 + 15) / 16 * 16 + (size_t)p.cap * sizeof(Cand);
    const size_t lds = merge > BLOCKS * sizeof(u64) ? merge : BLOCKS * sizeof(u64);
    const dim3 grid(a.batch * p.lists);
    if (fp32)
        hipLaunchKernelGGL((beam_select_kernel<float>), grid, dim3(SEL_THREADS), lds, st, static_cast<const float*>(logits), a, p);
    else
        hipLaunchKernelGGL((beam_select_kernel<_Float16>), grid, dim3(SEL_THREADS), lds, st,
                           static_cast<const _Float16*>(logits), a, p);
    return hipGetLastError();
}

// dst[o][b * out_beams + j][i][:] = src[o][b * beams + parents[b][j]][i][:], pieces of p.bytes bytes at byte strides.
// A workgroup takes a part of one piece (o, row, i), `part` elements of V; pieces whose parent lies outside the beams are left alone.
template <typename V>
__global__ __launch_bounds__(256) void beam_reorder_kernel(const char* src, const int64_t* parents, char* dst, ReorderArgs p, long part)
{
    const long rows = (long)p.batch * p.out_beams;
    const long length = p.bytes / (long)sizeof(V), parts = (length + part - 1) / part;
    for (long u = blockIdx.x; u < p.outer * rows * p.inner * parts; u += gridDim.x) {
        const long q = u / parts, c0 = u % parts * part;
        const long i = q % p.inner, r = q / p.inner % rows, o = q / p.inner / rows;
        const int64_t parent = parents[r];
        if (parent < 0 || parent >= p.beams) continue;
        const char* s = src + o * p.src[0] + (r / p.out_beams * p.beams + parent) * p.src[1] + i * p.src[2];
        char* d = dst + o * p.dst[0] + r * p.dst[1] + i * p.dst[2];
        for (long c = c0 + threadIdx.x; c < min(c0 + part, length); c += 256)
            reinterpret_cast<V*>(d)[c] = reinterpret_cast<const V*>(s)[c];
    }
}

namespace {

// Few large pieces are divided among workgroups, 8 per CU in all, into no less than one access per thread: 4 pieces of 64 MiB 111 us, 4.9
// TB/s, undivided 6980; 32 of 8 MiB 110 and 920.  A cache's pieces (42 layers of 32 rows, a
// sequence's 8 having 5.25 distinct parents in the mean: 1.02 GB to read once, 1.55 to write) 551 us, 4.65 TB/s.
template <typename V>
hipError_t reorder_launch(const char* src, const int64_t* parents, char* dst, const ReorderArgs& p, hipStream_t st)
{
    constexpr long SLOTS = 2048;
    const long pieces = p.outer * p.batch * p.out_beams * p.inner, length = p.bytes / (long)sizeof(V);
    const long most = pieces < SLOTS ? (SLOTS + pieces - 1) / pieces : 1;
    const long part = ((length + most - 1) / most + 255) / 256 * 256, units = pieces * ((length + part - 1) / part);
    hipLaunchKernelGGL((beam_reorder_kernel<V>), dim3((unsigned)(units < 65536 ? units : 65536)), dim3(256), 0, st, src, parents,
                       dst, p, part);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_beam_reorder(const void* src, const int64_t* parents, void* dst, const ReorderArgs& p, hipStream_t st)
{
    if (p.outer == 0 || p.batch == 0 || p.out_beams == 0 || p.inner == 0 || p.bytes == 0) return hipSuccess;
    // the widest access that every piece's address and length allow
    uint64_t low = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | (uint64_t)p.bytes;
    for (int i = 0; i < 3; ++i) low |= (uint64_t)p.src[i] | (uint64_t)p.dst[i];
    const char* s = static_cast<const char*>(src);
    char* d = static_cast<char*>(dst);
    return low % 16 == 0  ? reorder_launch<hx_u4>(s, parents, d, p, st)
           : low % 4 == 0 ? reorder_launch<uint32_t>(s, parents, d, p, st)
           : low % 2 == 0 ? reorder_launch<uint16_t>(s, parents, d, p, st)
                          : reorder_launch<uint8_t>(s, parents, d, p, st);
}

}  // namespace hx
