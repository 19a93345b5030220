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
// Selection is one launch.  A workgroup takes one chunk of one row: it reads the chunk once into registers, and from there
// come the chunk's maximum, the sum of its exponentials and its n largest logits.  The last workgroup of a sequence to
// arrive merges the chunks: the rows' log-sum-exp in 64 bits, the candidates' scores in 64 bits, the n best of them.
//
// The n largest of a set spread over threads, without sorting it: the n-th largest of the threads' maxima is a lower bound of
// the n-th largest of all, and only elements that reach it (n to 2n of random ones) are ranked against each other.  Sets with more
// ties at that bound than the candidate buffer holds are picked one by one instead.
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

// The n-th largest of 64 P keys in LDS, for one wave (0 where fewer than n are above 0): the key's bits from the top, each kept if
// n keys still reach the value.
template <int P>
HX_INLINE uint32_t nth_largest(const uint32_t* keys, int n)
{
    const int lane = threadIdx.x & 63;
    uint32_t k[P];
#pragma unroll
    for (int p = 0; p < P; ++p) k[p] = keys[64 * p + lane];
    uint32_t t = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = t | (1u << bit);
        int count = 0;
#pragma unroll
        for (int p = 0; p < P; ++p) count += __popcll(__ballot(k[p] >= c));
        if (count >= n) t = c;
    }
    return t;
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
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t t = n <= 32 ? nth_largest<1>(keys, n) : nth_largest<4>(keys, n);
        if (threadIdx.x == 0) bound = t;
    }
    __syncthreads();
    return bound;
}

HX_INLINE float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
HX_INLINE float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

struct BeamPlan {
    int chunks, lists;         // chunks of a row; beams * chunks, the lists of a sequence
    FastDiv by_chunks, by_lists;
    int cap;                   // candidates (16 bytes) that the LDS buffer holds
    u64* entries;              // [batch][n][lists]: the r-th best of each list, key << 32 | ~token, 0: none
    float2* stats;             // [batch][lists]: the chunk's maximum, the sum of exp(logit - maximum)
    int* counters;             // arrivals per sequence
};

constexpr int SEL_THREADS = 256;
constexpr int MERGE_E = 16;                         // candidates of a thread in one round of the merge
constexpr int MERGE = SEL_THREADS * MERGE_E;        // and of the workgroup

// A candidate of the merge: its score (-inf: none) and w * vocab + token.
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

// One chunk of SEL_THREADS * E logits of row w of sequence b, as list `list` of the sequence.
template <typename T, int E>
HX_INLINE void select_chunk(const T* x, int chunk, int list, const BeamArgs& a, const BeamPlan& p, long b, char* lds)
{
    constexpr int VEC = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
    __shared__ uint32_t keys[SEL_THREADS];
    __shared__ float part[2][4];
    __shared__ int count;
    u64* cand = reinterpret_cast<u64*>(lds);
    const int cap = 2 * p.cap;  // entries of 8 bytes
    const int tid = threadIdx.x, wave = tid >> 6;
    const int base = chunk * (SEL_THREADS * E), room = a.vocab - base;  // logits from the chunk's start to the row's end
    float v[E];
    if (room >= SEL_THREADS * E) {
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const vec t = *reinterpret_cast<const vec*>(x + base + (i * SEL_THREADS + tid) * VEC);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i * VEC + j] = (float)t[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int o = (i * SEL_THREADS + tid) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i * VEC + j] = -INFINITY;
            if (o + VEC <= room) {
                const vec t = *reinterpret_cast<const vec*>(x + base + o);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[i * VEC + j] = (float)t[j];
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (o + j < room) v[i * VEC + j] = (float)x[base + o + j];
            }
        }
    }
    float most = -INFINITY;  // a NaN is skipped here and makes the sum a NaN below
#pragma unroll
    for (int i = 0; i < E; ++i) most = fmaxf(most, v[i]);
    const float wm = wave_max(most);
    if ((tid & 63) == 0) part[0][wave] = wm;
    if (tid == 0) count = 0;
    const uint32_t bound = bound_of(float_key(most), a.n, keys);  // its barriers publish part[0] and count
    const float top = fmaxf(fmaxf(part[0][0], part[0][1]), fmaxf(part[0][2], part[0][3]));
    // elements that reach the bound
    if (float_key(most) >= bound && most > -INFINITY) {
        const float least = bound > KEY_NEG_INF ? key_float(bound) : -INFINITY;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (v[i] >= least && v[i] > -INFINITY) {
                const int at = atomicAdd(&count, 1);
                const uint32_t token = base + (i / VEC * SEL_THREADS + tid) * VEC + i % VEC;
                if (at < cap) cand[at] = (u64)float_key(v[i]) << 32 | (uint32_t)~token;
            }
    }
    // exp of the exact difference to the maximum (0 in its place in a chunk of -inf, whose sum is 0)
    const float sub = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) sum += __builtin_amdgcn_exp2f((v[i] - sub) * 1.44269504f);
    sum = wave_sum(sum);
    if ((tid & 63) == 0) part[1][wave] = sum;
    __syncthreads();
    const int c = count;
    const __amdgpu_buffer_rsrc_t out = coherent_rsrc(p.entries + (size_t)b * a.n * p.lists + list);
    if (c <= cap) {
        for (int i = tid; i < c; i += SEL_THREADS) {
            const u64 mine = cand[i];
            int r = 0;
            for (int j = 0; j < c; ++j) r += cand[j] > mine;
            if (r < a.n) coherent_store8(out, r * p.lists * 8, mine);
        }
        for (int r = c + tid; r < a.n; r += SEL_THREADS) coherent_store8(out, r * p.lists * 8, 0);
    } else {  // more ties than the buffer holds: one after the other
        u64* best = cand;  // [4]
        u64 last = ~0ull;
        for (int r = 0; r < a.n; ++r) {
            u64 m = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const uint32_t token = base + (i / VEC * SEL_THREADS + tid) * VEC + i % VEC;
                const u64 k = v[i] > -INFINITY ? (u64)float_key(v[i]) << 32 | (uint32_t)~token : 0;
                if (k < last && k > m) m = k;
            }
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) {
                const u64 q = __shfl_xor(m, o, 64);
                m = q > m ? q : m;
            }
            __syncthreads();  // every thread is done with the buffer
            if ((tid & 63) == 0) best[wave] = m;
            __syncthreads();
            const u64 h = best[0] > best[1] ? best[0] : best[1], g = best[2] > best[3] ? best[2] : best[3];
            last = h > g ? h : g;
            if (tid == 0) coherent_store8(out, r * p.lists * 8, last);
        }
    }
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
    __shared__ int count;
    double* offset = reinterpret_cast<double*>(lds);
    float* tops = reinterpret_cast<float*>(offset + a.beams);
    Cand* cand = reinterpret_cast<Cand*>(lds + ((size_t)a.beams * 12 + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 63, n = a.n;
    const __amdgpu_buffer_rsrc_t rs = coherent_rsrc(p.stats + (size_t)b * p.lists);
    const __amdgpu_buffer_rsrc_t re = coherent_rsrc(p.entries + (size_t)b * n * p.lists);
    // score = offset[w] + (logit - tops[w]); offset NaN: the row has no candidates
    for (int w = tid >> 6; w < a.beams; w += 4) {
        const double cum = (double)a.cum[b * a.beams + w];
        double off = NAN;
        float top = 0.0f;
        if (!(fabs(cum) < INFINITY)) {
        } else if (a.done && a.done[b * a.beams + w]) {
            off = cum;
        } else {
            float m = -INFINITY;
            for (int c = lane; c < p.chunks; c += 64)
                m = fmaxf(m, __builtin_bit_cast(float2, coherent_load8(rs, (w * p.chunks + c) * 8)).x);
            m = wave_max(m);
            double s = 0.0;
            for (int c = lane; c < p.chunks; c += 64) {
                const float2 st = __builtin_bit_cast(float2, coherent_load8(rs, (w * p.chunks + c) * 8));
                s += (double)st.y * exp((double)st.x - (double)m);
            }
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
            if (fabsf(m) < INFINITY && s < INFINITY) off = cum - log(s), top = m;  // a NaN fails both tests
        }
        if (lane == 0) offset[w] = off, tops[w] = top;
    }
    const int total = n * p.lists;
    int kept = 0;  // entries of carry
    __syncthreads();
    for (int done = 0; done < total;) {
        const int fresh = min(total - done, MERGE - kept);
        Cand v[MERGE_E];
        u64 e[MERGE_E];
#pragma unroll
        for (int i = 0; i < MERGE_E; ++i) {
            const int q = i * SEL_THREADS + tid;
            e[i] = q < fresh ? coherent_load8(re, (done + q) * 8) : 0;
        }
        double most = -INFINITY;
#pragma unroll
        for (int i = 0; i < MERGE_E; ++i) {
            const int q = i * SEL_THREADS + tid;
            v[i] = {-INFINITY, 0};
            if (q < fresh) {
                const uint32_t at = done + q, rank = div_by(at, p.by_lists), list = at - rank * p.lists;
                const uint32_t w = div_by(list, p.by_chunks);
                const double off = offset[w];
                const bool fin = a.done && a.done[b * a.beams + w];
                if (off == off) {
                    if (fin) {
                        if (rank == 0 && list == w * p.chunks) v[i] = {off, w * (u64)a.vocab + a.eos};
                    } else if (e[i]) {
                        v[i] = {off + ((double)key_float((uint32_t)(e[i] >> 32)) - (double)tops[w]),
                                w * (u64)a.vocab + (uint32_t)~(uint32_t)e[i]};
                    }
                }
            } else if (q < fresh + kept) {
                v[i] = carry[q - fresh];
            }
            most = fmax(most, v[i].s);
        }
        if (tid == 0) count = 0;
        // scores rounded to fp32 keep their order (not strictly): the bound holds for the rounded ones
        const uint32_t bound = bound_of(most > -INFINITY ? float_key((float)most) : 0, n, keys);
        if (most > -INFINITY && float_key((float)most) >= bound) {
#pragma unroll
            for (int i = 0; i < MERGE_E; ++i)
                if (v[i].s > -INFINITY && float_key((float)v[i].s) >= bound) {
                    const int at = atomicAdd(&count, 1);
                    if (at < p.cap) cand[at] = v[i];
                }
        }
        __syncthreads();
        const int c = count;
        if (c <= p.cap) {
            for (int i = tid; i < c; i += SEL_THREADS) {
                const Cand mine = cand[i];
                int r = 0;
                for (int j = 0; j < c; ++j) r += better(cand[j].s, cand[j].at, mine.s, mine.at);
                if (r < n) carry[r] = mine;
            }
            kept = min(c, n);
            __syncthreads();
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
                    const u64 at = __shfl_xor(m.at, o, 64);
                    if (better(s, at, m.s, m.at)) m = {s, at};
                }
                if (lane == 0) best[tid >> 6] = m;
                __syncthreads();
                last = best[0];
                for (int i = 1; i < 4; ++i)
                    if (better(best[i].s, best[i].at, last.s, last.at)) last = best[i];
                if (tid == 0) carry[r] = last;
                __syncthreads();
            }
            kept = n;
        }
        done += fresh;
    }
    for (int r = tid; r < n; r += SEL_THREADS) {
        const bool found = r < kept;
        const u64 at = found ? carry[r].at : 0;
        a.scores[b * n + r] = found ? (float)carry[r].s : -INFINITY;
        a.parents[b * n + r] = found ? (int64_t)(at / a.vocab) : -1;
        a.tokens[b * n + r] = found ? (int64_t)(at % a.vocab) : -1;
    }
}

}  // namespace

// grid: [batch][beams][chunks]
template <typename T, int E>
__global__ __launch_bounds__(SEL_THREADS) void beam_select_kernel(const T* logits, BeamArgs a, BeamPlan p)
{
    extern __shared__ __align__(16) char beam_lds[];
    const uint32_t row = div_by(blockIdx.x, p.by_chunks), chunk = blockIdx.x - row * p.chunks;
    const uint32_t b = div_by(blockIdx.x, p.by_lists), list = blockIdx.x - b * p.lists;
    // rows that are finished or dead are not read
    if (!(a.done && a.done[row]) && fabsf(a.cum[row]) < INFINITY)
        select_chunk<T, E>(logits + row * a.ld, chunk, list, a, p, b, beam_lds);
    if (!arrive_last(p.counters + b, p.lists)) return;
    select_merge(a, p, b, beam_lds);
}

namespace {

// Logits of a chunk: 8192 (32 per thread), or 2048 where that leaves fewer than 4 workgroups per CU.
int select_elems(long rows, int vocab) { return rows * ((vocab + 8191) / 8192) >= 1024 ? 32 : 8; }

struct SelectLayout {
    int elems;
    long chunks, lists;
    size_t entries, stats, total;  // bytes
    SelectLayout(int batch, int beams, int vocab, int n)
    {
        elems = select_elems((long)batch * beams, vocab);
        chunks = ((long)vocab + SEL_THREADS * elems - 1) / (SEL_THREADS * elems);
        lists = beams * chunks;
        entries = (size_t)batch * n * lists * sizeof(u64);
        stats = (size_t)batch * lists * sizeof(float2);
        total = HX_COUNTER_BYTES + entries + stats;
    }
};

FastDiv fast_div(uint32_t d) { return {d, (uint32_t)(((1ull << 32) + d - 1) / d)}; }

template <typename T, int E>
hipError_t select_launch(const void* logits, const BeamArgs& a, const BeamPlan& p, size_t lds, hipStream_t st)
{
    hipLaunchKernelGGL((beam_select_kernel<T, E>), dim3(a.batch * p.lists), dim3(SEL_THREADS), lds, st,
                       static_cast<const T*>(logits), a, p);
    return hipGetLastError();
}

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
    // the candidate buffer, 16 times what is asked for (32 times in a chunk's 8-byte entries): ties aside the bound is reached by
    // n threads (or quads) at most, each with at most 32 elements or MERGE_E candidates, and by n to 2n elements as a rule
    const BeamPlan p{(int)l.chunks, (int)l.lists, fast_div(l.chunks), fast_div(l.lists), a.n * MERGE_E,
                     reinterpret_cast<u64*>(base + HX_COUNTER_BYTES),
                     reinterpret_cast<float2*>(base + HX_COUNTER_BYTES + l.entries), reinterpret_cast<int*>(base)};
    const size_t lds = ((size_t)a.beams * 12 + 15) / 16 * 16 + (size_t)p.cap * sizeof(Cand);
    if (l.elems == 32)
        return fp32 ? select_launch<float, 32>(logits, a, p, lds, st) : select_launch<_Float16, 32>(logits, a, p, lds, st);
    return fp32 ? select_launch<float, 8>(logits, a, p, lds, st) : select_launch<_Float16, 8>(logits, a, p, lds, st);
}

// dst[o][b * out_beams + j][i][:] = src[o][b * beams + parents[b][j]][i][:], pieces of p.bytes bytes at byte strides.
// A workgroup takes one piece (o, row, i); pieces whose parent lies outside the beams are left alone.
template <typename V>
__global__ __launch_bounds__(256) void beam_reorder_kernel(const char* src, const int64_t* parents, char* dst, ReorderArgs p)
{
    const long rows = (long)p.batch * p.out_beams;
    for (long q = blockIdx.x; q < p.outer * rows * p.inner; q += gridDim.x) {
        const long i = q % p.inner, r = q / p.inner % rows, o = q / p.inner / rows;
        const int64_t parent = parents[r];
        if (parent < 0 || parent >= p.beams) continue;
        const char* s = src + o * p.src[0] + (r / p.out_beams * p.beams + parent) * p.src[1] + i * p.src[2];
        char* d = dst + o * p.dst[0] + r * p.dst[1] + i * p.dst[2];
        for (long c = threadIdx.x; c < p.bytes / (long)sizeof(V); c += 256)
            reinterpret_cast<V*>(d)[c] = reinterpret_cast<const V*>(s)[c];
    }
}

hipError_t launch_beam_reorder(const void* src, const int64_t* parents, void* dst, const ReorderArgs& p, hipStream_t st)
{
    const long pieces = p.outer * p.batch * p.out_beams * p.inner;
    if (pieces == 0 || p.bytes == 0) return hipSuccess;
    // the widest access that every piece's address and length allow
    uint64_t low = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | (uint64_t)p.bytes;
    for (int i = 0; i < 3; ++i) low |= (uint64_t)p.src[i] | (uint64_t)p.dst[i];
    const dim3 grid((unsigned)(pieces < 65536 ? pieces : 65536));
    const char* s = static_cast<const char*>(src);
    char* d = static_cast<char*>(dst);
    if (low % 16 == 0) hipLaunchKernelGGL((beam_reorder_kernel<hx_u4>), grid, dim3(256), 0, st, s, parents, d, p);
    else if (low % 4 == 0) hipLaunchKernelGGL((beam_reorder_kernel<uint32_t>), grid, dim3(256), 0, st, s, parents, d, p);
    else if (low % 2 == 0) hipLaunchKernelGGL((beam_reorder_kernel<uint16_t>), grid, dim3(256), 0, st, s, parents, d, p);
    else hipLaunchKernelGGL((beam_reorder_kernel<uint8_t>), grid, dim3(256), 0, st, s, parents, d, p);
    return hipGetLastError();
}

}  // namespace hx
