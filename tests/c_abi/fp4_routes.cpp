// Where the expert layer for a few tokens finds its routes (frx_policy.hpp), as a shared library for
// tests/test_fp4_routes.py. Built with g++; no GPU.
#include "frx_policy.hpp"

extern "C" int fp4_routes_inside_of(uint32_t T) { return frx::fp4_routes_inside(T); }
