// The 4-bit linears' kernel rules (frx_policy.hpp) as a shared library for
// tests/test_fp4_plan.py. Built with g++; no GPU.
#include "frx_policy.hpp"

extern "C" void fp4_plan_of(uint32_t M, uint32_t K, uint32_t N, int cus, int out[3]) {
  const frx::Fp4Plan p = frx::fp4_plan(M, K, N, cus);
  out[0] = p.tile;
  out[1] = p.S;
  out[2] = p.per;
}

extern "C" int fp4_grouped_tile_of(uint32_t R, uint32_t K, uint32_t N, uint32_t E, int cus) {
  return frx::fp4_grouped_tile(R, K, N, E, cus);
}

extern "C" int fp4_grad_tile_of(uint32_t R, uint32_t N, uint32_t K, uint32_t E, int cus) {
  return frx::fp4_grad_tile(R, N, K, E, cus);
}

// gate and up (planes of x) and down (planes of h): steps, tiles, slices, steps of a slice.
extern "C" void fp4_few_of(uint32_t T, uint32_t K, uint32_t E, uint32_t top_k, int planes, int down, int out[4]) {
  const frx::Fp4FewPlan p = down ? frx::fp4_down_plan(T, K, E, top_k, planes) : frx::fp4_gate_up_plan(T, K, E, top_k, planes);
  out[0] = p.steps;
  out[1] = p.tiles;
  out[2] = p.slices;
  out[3] = p.per;
}
