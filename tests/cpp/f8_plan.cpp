// The plan of the 8-bit linear and its gated pair (csrc/hx_f8_plan.hpp) for tests/test_f8_plan.py.
#include "hx_f8_plan.hpp"

extern "C" {

void f8_plan(int M, int N, int K, int sums, int split, long out[6])
{
    const hx::F8Plan p = hx::f8_plan(M, N, K, (hx::F8Sums)sums, split != 0);
    const long v[6] = {(long)p.kind, p.splits, p.steps, p.tiles, (long)p.partial, (long)p.products};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
}
size_t f8_call_workspace(int M, int N, int K, int sums) { return hx::f8_call_workspace(M, N, K, (hx::F8Sums)sums); }
int f8_most_rows(int N, int pair) { return hx::f8_most_rows(N, pair != 0); }
void f8_tile(int sums, int kind, int out[3])
{
    const hx::F8Tile& t = hx::F8_TILES[sums][kind];
    out[0] = t.bn, out[1] = t.bm, out[2] = t.part != 0.f;
}

}  // extern "C"
