// Test-only: the host side of csrc/tile.hpp -- which tiles and splits a product takes, and what
// a launch refuses -- with the stand-in of the HIP runtime.  Its kernel never runs.
#include "../../thrml-rs_amd/csrc/tile.hpp"

namespace thrml {
static std::string last_error;
void set_error(const std::string &msg) { last_error = msg; }
int fail(int code, const std::string &msg) {
  last_error = msg;
  return code;
}
int hip_fail(hipError_t, const char *what) { return fail(THRML_EHIP, what); }
}  // namespace thrml

struct Grid {
  uint32_t ta, tb, splits, steps;
};
__global__ void nothing(Grid) {}

// kinds: n of {na, nb, kb}, with their times; plan: kind, ta, tb, splits, steps
extern "C" void tile_plan(const uint32_t *kinds, const float *times, int n, uint64_t cols, uint64_t rows, int halves, uint64_t row_bytes,
                          uint64_t out_values, uint32_t *plan) {
  thrml::TileKind k[8];
  for (int i = 0; i < n; ++i) k[i] = {kinds[3 * i], kinds[3 * i + 1], kinds[3 * i + 2], times[2 * i], times[2 * i + 1]};
  static thrml_ctx ctx;
  const thrml::TilePlan p = thrml::plan_tiles(&ctx, k, n, cols, rows, halves != 0, row_bytes, out_values);
  plan[0] = (uint32_t)p.kind;
  plan[1] = p.ta;
  plan[2] = p.tb;
  plan[3] = p.splits;
  plan[4] = p.steps;
}

extern "C" int tile_launch(uint32_t ta, uint32_t tb, uint32_t splits, uint32_t steps) {
  static thrml_ctx ctx;
  return thrml::launch_tiles(&ctx, &nothing, Grid{ta, tb, splits, steps}, 256, 0);
}
extern "C" const char *tile_error() { return thrml::last_error.c_str(); }
