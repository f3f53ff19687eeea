// The 8-bit linears' kernel rules (frx_policy.hpp) as a shared library for
// tests/test_fp8_plan.py. Built with g++; no GPU.
#include "frx_policy.hpp"

extern "C" void fp8_plan_of(uint32_t M, uint32_t K, uint32_t N, int b_rows, int pipe8, int cus, int out[3]) {
  const frx::Fp8Plan p = frx::fp8_plan(M, K, N, b_rows, pipe8, cus);
  out[0] = p.tile;
  out[1] = p.S;
  out[2] = p.per;
}

extern "C" int fp8_grouped_tile_of(uint32_t R, uint32_t N, uint32_t E, int pipe8, int cus) {
  return frx::fp8_grouped_tile(R, N, E, pipe8, cus);
}
