// hx_beam.hip -- one step of beam search on gfx950: the best continuations over beams and vocabulary, and the surviving
// beams' states.
//
//   score(w, v) = cum[w] + (logit[w][v] - logsumexp_v logit[w]),  the n best of each sequence in descending order,
//   the lowest w * vocab + v first among equals
//
// A finished beam (done[w] != 0) has one candidate, (w, eos) with score cum[w].  A beam whose cum is not finite, whose logits
// hold a NaN or +inf, or are all -inf, has none (its log-softmax is not defined); a logit of -inf is no candidate.
// Sequences with fewer than n candidates get score -inf, parent -1 and token -1 behind them.
#include "hx_device.hpp"
#include "hx_kernels.hpp"

namespace hx {

namespace {

// Sums over a workgroup of 256 threads, in a fixed order; every thread gets the result.
template <typename T, typename F>
HX_INLINE T block_reduce(T v, F op, T* lds)
{
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int h = 128; h >= 1; h >>= 1) {
        if ((int)threadIdx.x < h) lds[threadIdx.x] = op(lds[threadIdx.x], lds[threadIdx.x + h]);
        __syncthreads();
    }
    v = lds[0];
    __syncthreads();
    return v;
}

}  // namespace

// offset[row] = (max of the row, cum - log of the sum of exp(logit - max)), NaN for a row without candidates.
template <typename T>
__global__ __launch_bounds__(256) void beam_lse_kernel(const T* logits, BeamArgs a, double2* offset)
{
    __shared__ double lds[256];
    const long row = blockIdx.x;
    const T* x = logits + row * a.ld;
    double top = -INFINITY;
    bool bad = false;
    for (int v = threadIdx.x; v < a.vocab; v += 256) {
        const double l = (double)x[v];
        bad |= l != l;
        top = fmax(top, l);
    }
    top = block_reduce(top, [](double p, double q) { return fmax(p, q); }, lds);
    bad = block_reduce(bad ? 1.0 : 0.0, [](double p, double q) { return fmax(p, q); }, lds) != 0.0;
    double sum = 0.0;
    for (int v = threadIdx.x; v < a.vocab; v += 256) sum += exp((double)x[v] - top);
    sum = block_reduce(sum, [](double p, double q) { return p + q; }, lds);
    if (threadIdx.x == 0) {
        const double c = (double)a.cum[row];
        const bool none = bad || !(fabs(top) < INFINITY) || !(fabs(c) < INFINITY);
        offset[row] = none ? double2{0.0, (double)NAN} : double2{top, c - log(sum)};
    }
}

// One workgroup per sequence: n rounds, each taking the best candidate that comes after the last one taken.
template <typename T>
__global__ __launch_bounds__(256) void beam_pick_kernel(const T* logits, BeamArgs a, const double2* offset)
{
    __shared__ double best_s[256];
    __shared__ long best_i[256];
    const long b = blockIdx.x;
    double last = INFINITY;
    long last_i = -1;
    const long none = 0x7fffffffffffffffL;
    for (int r = 0; r < a.n; ++r) {
        double s = -INFINITY;
        long at = none;
        for (long i = threadIdx.x; i < (long)a.beams * a.vocab; i += 256) {
            const long w = b * a.beams + i / a.vocab, v = i % a.vocab;
            double c;
            if (a.done && a.done[w]) {
                c = v == a.eos ? (double)a.cum[w] : -INFINITY;
                if (!(fabs(c) < INFINITY)) continue;
            } else {
                c = ((double)logits[w * a.ld + v] - offset[w].x) + offset[w].y;
                if (!(fabs(c) < INFINITY)) continue;
            }
            if (!(c < last || (c == last && i > last_i))) continue;
            if (c > s || (c == s && i < at)) s = c, at = i;
        }
        best_s[threadIdx.x] = s;
        best_i[threadIdx.x] = at;
        __syncthreads();
        for (int h = 128; h >= 1; h >>= 1) {
            const int t = threadIdx.x, u = t + h;
            if (t < h && (best_s[u] > best_s[t] || (best_s[u] == best_s[t] && best_i[u] < best_i[t])))
                best_s[t] = best_s[u], best_i[t] = best_i[u];
            __syncthreads();
        }
        last = best_s[0], last_i = best_i[0];
        __syncthreads();
        if (threadIdx.x == 0) {
            const bool found = last_i != none;
            a.scores[b * a.n + r] = found ? (float)last : -INFINITY;
            a.parents[b * a.n + r] = found ? last_i / a.vocab : -1;
            a.tokens[b * a.n + r] = found ? last_i % a.vocab : -1;
        }
    }
}

size_t beam_select_workspace_bytes(int batch, int beams, int vocab, int n)
{
    return HX_COUNTER_BYTES + (size_t)batch * beams * sizeof(double2);
}

template <typename T>
static hipError_t select_typed(const T* logits, const BeamArgs& a, void* ws, hipStream_t st)
{
    double2* offset = reinterpret_cast<double2*>(static_cast<char*>(ws) + HX_COUNTER_BYTES);
    hipLaunchKernelGGL((beam_lse_kernel<T>), dim3(a.batch * a.beams), dim3(256), 0, st, logits, a, offset);
    hipLaunchKernelGGL((beam_pick_kernel<T>), dim3(a.batch), dim3(256), 0, st, logits, a, offset);
    return hipGetLastError();
}

hipError_t launch_beam_select(const void* logits, bool fp32, const BeamArgs& a, void* ws, hipStream_t st)
{
    if (a.batch <= 0) return hipSuccess;
    return fp32 ? select_typed(static_cast<const float*>(logits), a, ws, st)
                : select_typed(static_cast<const _Float16*>(logits), a, ws, st);
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
