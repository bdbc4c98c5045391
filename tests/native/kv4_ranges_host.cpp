// CPU harness for how vqx_kv4_attention.hip cuts a call up: the plan that sizes the
// workspace and the ranges that its kernels work out of lengths and offsets, the
// same code on the host.  Kernels are turned into plain device functions, of which
// the host's pass makes no code.  Test-only.
#include <hip/hip_runtime.h>

#undef __global__
#define __global__ __device__
#undef __launch_bounds__
#define __launch_bounds__(...)
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(...) ((void)0)

#include "vqx_kv4_attention.hip"

namespace vqx {
int set_error(int code, const char*, ...) { return code; }
int check_launch(const char*) { return kOk; }
int num_cus() { return 256; }
}  // namespace vqx

extern "C" {

// Of one call: plan[4] (rows of a tile, tiles, tokens of a split, splits), and for
// every tile of every sequence lo, hi and the splits that the join adds up.
int vqx_host_kv4_ranges(int64_t room, int seqs, int kv, int dim, int group, int dtype, int n, const int32_t* cu, int most,
                        int window, int tree, const int32_t* lengths, int32_t* plan, int32_t* ranges) {
  using namespace vqx;
  Kv4View c = {};
  c.lengths = lengths, c.cap = (uint32_t)room, c.size = (uint32_t)room, c.seqs = (uint32_t)seqs, c.kv = (uint32_t)kv;
  Kv4Query q = {};
  const int64_t mask = 0;
  q.tokens = Kv4Tokens{cu, n, 0};
  q.heads = kv * group, q.group = group, q.most = most, q.window = window;
  q.tree = tree ? &mask : nullptr;
  const Kv4Plan p = kv4_plan(c, dim, q, dtype);
  plan[0] = p.rows, plan[1] = p.tiles, plan[2] = p.chunk, plan[3] = p.splits;
  const int step = p.rows == kRows ? kStep : kBlockStep;
  for (int b = 0; b < seqs; ++b)
    for (int t = 0; t < p.tiles; ++t, ranges += 3) {
      const TileRows r = tree ? tile_rows<true>(c, q, (uint32_t)b, t, p.rows, step) : tile_rows(c, q, (uint32_t)b, t, p.rows, step);
      ranges[0] = r.lo, ranges[1] = r.hi, ranges[2] = t * p.rows < r.rows ? joined_splits(r, p) : 0;
    }
  return 0;
}
}
