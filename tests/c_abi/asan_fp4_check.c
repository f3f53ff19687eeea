/* The 4-bit linears' and their expert layer's entry points as C declares them,
 * with the host code (frx_api.cpp) under AddressSanitizer and UBSan:
 *
 *  - Their signatures.
 *  - Every one with a null context returns FRX_ERR_DEVICE.
 *  - With "--device" (a GPU present) every argument check on a real context:
 *    null pointers, empty and oversized shapes, strides, alignments, types,
 *    experts, host arrays of exactly E entries on the heap, and the forced
 *    status. All are rejected before a launch; the pointers are device memory
 *    all the same. Then which calls need a workspace.
 * Prints "asan_fp4_check ok" and exits 0 when every check passes. */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "frx_ternary.h"

static int failures = 0;
#define EXPECT(cond)                                                       \
  do {                                                                     \
    if (!(cond)) {                                                         \
      fprintf(stderr, "%s:%d: expected %s\n", __FILE__, __LINE__, #cond); \
      failures++;                                                          \
    }                                                                      \
  } while (0)

/* signatures */
static frx_status (*const quantize)(frx_ctx *, const void *, frx_dtype, uint32_t, uint32_t, size_t, frx_fp4_blocks,
                                    uint8_t *, size_t, uint8_t *) = frx_fp4_quantize;
static frx_status (*const dequantize)(frx_ctx *, const uint8_t *, size_t, const uint8_t *, uint32_t, uint32_t, void *,
                                      frx_dtype, size_t) = frx_fp4_dequantize;
static frx_status (*const linear)(frx_ctx *, const uint8_t *, size_t, const uint8_t *, const uint8_t *, size_t,
                                  const uint8_t *, void *, frx_dtype, uint32_t, uint32_t, uint32_t) = frx_fp4_linear;
static frx_status (*const act)(frx_ctx *, const void *, frx_dtype, const uint8_t *, size_t, const uint8_t *, void *,
                               frx_dtype, uint32_t, uint32_t, uint32_t) = frx_fp4_linear_act;
static frx_status (*const grouped)(frx_ctx *, const uint8_t *, size_t, const uint8_t *, const uint8_t *const *, size_t,
                                   const uint8_t *const *, const uint32_t *, uint32_t, void *, frx_dtype, uint32_t,
                                   uint32_t, uint32_t) = frx_fp4_linear_grouped;
static frx_status (*const grad)(frx_ctx *, const uint8_t *, size_t, const uint8_t *, const uint8_t *, size_t,
                                const uint8_t *, const uint32_t *, uint32_t, void *const *, frx_dtype, uint32_t, uint32_t,
                                uint32_t) = frx_fp4_grad_weight_grouped;
static frx_status (*const ffn)(frx_ctx *, const void *, frx_dtype, const void *, frx_dtype, const uint8_t *const *,
                               const uint8_t *const *, const uint8_t *const *, const uint8_t *const *,
                               const uint8_t *const *, const uint8_t *const *, uint32_t, uint32_t, uint32_t, uint32_t,
                               uint32_t, frx_activation, void *, frx_dtype, uint32_t *, float *) = frx_fp4_moe_ffn;

static void check_host(void) {
  const frx_status D = FRX_ERR_DEVICE;
  EXPECT(quantize(NULL, NULL, FRX_F32, 1, 1, 1, FRX_FP4_ROWS, NULL, 16, NULL) == D);
  EXPECT(dequantize(NULL, NULL, 16, NULL, 1, 1, NULL, FRX_F32, 1) == D);
  EXPECT(linear(NULL, NULL, 16, NULL, NULL, 16, NULL, NULL, FRX_F32, 1, 32, 1) == D);
  EXPECT(act(NULL, NULL, FRX_F32, NULL, 16, NULL, NULL, FRX_F32, 1, 32, 1) == D);
  EXPECT(grouped(NULL, NULL, 16, NULL, NULL, 16, NULL, NULL, 1, NULL, FRX_F32, 1, 32, 1) == D);
  EXPECT(grad(NULL, NULL, 16, NULL, NULL, 16, NULL, NULL, 1, NULL, FRX_F32, 32, 1, 1) == D);
  EXPECT(ffn(NULL, NULL, FRX_F32, NULL, FRX_F32, NULL, NULL, NULL, NULL, NULL, NULL, 1, 32, 32, 1, 1, FRX_ACT_SILU, NULL,
             FRX_F32, NULL, NULL) == D);
}

static void check_products(frx_ctx *c, void *mem) {
  const frx_status S = FRX_ERR_SHAPE, U = FRX_ERR_UNSUPPORTED;
  uint8_t *q = mem;
  float *f = mem;
  const uint32_t *o = mem;
  const size_t far = (size_t)1 << 22;
  /* the quantiser */
#define Q(x, xt, m, k, ldx, blocks, out, ldq, sc) \
  quantize(c, x, (frx_dtype)(xt), m, k, ldx, (frx_fp4_blocks)(blocks), out, ldq, sc)
  EXPECT(Q(NULL, 0, 2, 32, 32, 0, q, 16, q) == S && Q(f, 0, 2, 32, 32, 0, NULL, 16, q) == S);
  EXPECT(Q(f, 0, 2, 32, 32, 0, q, 16, NULL) == S);
  EXPECT(Q(f, 0, 0, 32, 32, 0, q, 16, q) == S && Q(f, 0, 2, 0, 32, 0, q, 16, q) == S);
  EXPECT(Q(f, 2, 2, 32, 32, 0, q, 16, q) == U && Q(f, 0, 2, 32, 32, 2, q, 16, q) == U);
  EXPECT(Q(f, 0, 2, 32, 31, 0, q, 16, q) == S && Q(f, 0, 2, 32, 32, 0, q, 24, q) == S);
  EXPECT(Q(f, 0, 2, 33, 33, 0, q, 16, q) == S && Q(f, 0, 33, 2, 2, 1, q, 16, q) == S);
  EXPECT(Q(q + 2, 0, 2, 32, 32, 0, q, 16, q) == S && Q(q + 1, 1, 2, 32, 32, 0, q, 16, q) == S);
  EXPECT(Q(f, 0, 2, 32, 32, 0, q + 8, 16, q) == S && Q(f, 0, 2, 32, 32, 0, q, 16, q + 2) == S);
  EXPECT(Q(f, 0, 0xFFFFFFFFu, 32, 32, 0, q, 16, q) == S && Q(f, 0, 1u << 30, 128, 128, 0, q, 64, q) == S);
  EXPECT(Q(f, 0, 1u << 20, 1u << 20, 1u << 20, 1, q, 1u << 19, q) == S);
  EXPECT(strlen(frx_last_error(c)) > 0);
  /* and back */
#define B(a, ldq, sc, m, k, y, yt, ldy) dequantize(c, a, ldq, sc, m, k, y, (frx_dtype)(yt), ldy)
  EXPECT(B(NULL, 16, q, 2, 32, f, 0, 32) == S && B(q, 16, NULL, 2, 32, f, 0, 32) == S && B(q, 16, q, 2, 32, NULL, 0, 32) == S);
  EXPECT(B(q, 16, q, 0, 32, f, 0, 32) == S && B(q, 16, q, 2, 0, f, 0, 32) == S && B(q, 16, q, 2, 32, f, 2, 32) == U);
  EXPECT(B(q, 24, q, 2, 32, f, 0, 32) == S && B(q, 16, q, 2, 33, f, 0, 33) == S && B(q, 16, q, 2, 32, f, 0, 31) == S);
  EXPECT(B(q + 8, 16, q, 2, 32, f, 0, 32) == S && B(q, 16, q + 2, 2, 32, f, 0, 32) == S);
  EXPECT(B(q, 16, q, 2, 32, q + 2, 0, 32) == S && B(q, 16, q, 2, 32, q + 1, 1, 32) == S);
  EXPECT(B(q, 16, q, 0xFFFFFFFFu, 32, f, 0, 32) == S);
  /* one product */
#define L(a, lda, sa, b, ldb, sb, y, yt, m, k, n) linear(c, a, lda, sa, b, ldb, sb, y, (frx_dtype)(yt), m, k, n)
  EXPECT(L(NULL, 16, q, q, 16, q, f, 0, 1, 32, 1) == S && L(q, 16, NULL, q, 16, q, f, 0, 1, 32, 1) == S);
  EXPECT(L(q, 16, q, NULL, 16, q, f, 0, 1, 32, 1) == S && L(q, 16, q, q, 16, NULL, f, 0, 1, 32, 1) == S);
  EXPECT(L(q, 16, q, q, 16, q, NULL, 0, 1, 32, 1) == S && L(q, 16, q, q, 16, q, f, 2, 1, 32, 1) == U);
  EXPECT(L(q, 16, q, q, 16, q, f, 0, 0, 32, 1) == S && L(q, 16, q, q, 16, q, f, 0, 1, 0, 1) == S);
  EXPECT(L(q, 16, q, q, 16, q, f, 0, 1, 32, 0) == S && L(q, 16, q, q, 16, q, f, 0, 1, 16, 1) == S);
  EXPECT(L(q, 32, q, q, 32, q, f, 0, 1, 48, 1) == S && L(q, 24, q, q, 16, q, f, 0, 1, 32, 1) == S);
  EXPECT(L(q, 16, q, q, 24, q, f, 0, 1, 32, 1) == S && L(q, 16, q, q, 32, q, f, 0, 1, 64, 1) == S);
  EXPECT(L(q, 32, q, q, 16, q, f, 0, 1, 64, 1) == S);
  EXPECT(L(q, far + 16, q, q, 16, q, f, 0, 1, 32, 1) == S && L(q, 16, q, q, far + 16, q, f, 0, 1, 32, 1) == S);
  EXPECT(L(q + 8, 16, q, q, 16, q, f, 0, 1, 32, 1) == S && L(q, 16, q, q + 8, 16, q, f, 0, 1, 32, 1) == S);
  EXPECT(L(q, 16, q + 2, q, 16, q, f, 0, 1, 32, 1) == S && L(q, 16, q, q, 16, q + 2, f, 0, 1, 32, 1) == S);
  EXPECT(L(q, 16, q, q, 16, q, q + 2, 0, 1, 32, 1) == S && L(q, 16, q, q, 16, q, q + 1, 1, 1, 32, 1) == S);
  EXPECT(L(q, 16, q, q, 16, q, f, 0, 0xFFFFFFFFu, 32, 1) == S && L(q, 16, q, q, 16, q, f, 0, 1, 32, 0xFFFFFFFFu) == S);
  EXPECT(L(q, 16, q, q, 16, q, f, 0, 1, 32, 1u << 27) == S && L(q, 16, q, q, 16, q, f, 0, 1u << 20, 32, 1u << 20) == S);
  /* with the activations quantised inside */
#define A(x, xt, b, ldb, sb, y, yt, m, k, n) act(c, x, (frx_dtype)(xt), b, ldb, sb, y, (frx_dtype)(yt), m, k, n)
  EXPECT(A(NULL, 0, q, 16, q, f, 0, 1, 32, 1) == S && A(f, 2, q, 16, q, f, 0, 1, 32, 1) == U);
  EXPECT(A(q + 2, 0, q, 16, q, f, 0, 1, 32, 1) == S && A(q + 1, 1, q, 16, q, f, 0, 1, 32, 1) == S);
  EXPECT(A(f, 0, NULL, 16, q, f, 0, 1, 32, 1) == S && A(f, 0, q, 16, NULL, f, 0, 1, 32, 1) == S);
  EXPECT(A(f, 0, q, 16, q, NULL, 0, 1, 32, 1) == S && A(f, 0, q, 16, q, f, 2, 1, 32, 1) == U);
  EXPECT(A(f, 0, q, 32, q, f, 0, 1, 48, 1) == S && A(f, 0, q, 24, q, f, 0, 1, 32, 1) == S);
  EXPECT(A(f, 0, q, 16, q, f, 0, 0, 32, 1) == S && A(f, 0, q, 16, q, f, 0, 1, 32, 0) == S);
  EXPECT(A(f, 0, q, 2 * far, q, f, 0, 1, 4 * (uint32_t)far, 1) == S);
  /* experts: host arrays of exactly E entries */
  enum { E = 3, N = 4, K = 32, R = 16 };
  const uint8_t **b = malloc(E * sizeof(*b)), **sb = malloc(E * sizeof(*sb));
  if (!b || !sb) abort();
  for (int e = 0; e < E; e++) b[e] = sb[e] = q;
#define G(a, lda, sa, bs, ldb, sbs, off, e, y, yt, r, k, n) \
  grouped(c, a, lda, sa, bs, ldb, sbs, off, e, y, (frx_dtype)(yt), r, k, n)
  EXPECT(G(q, 16, q, b, 16, sb, o, 0, f, 0, R, K, N) == S && G(q, 16, q, b, 16, sb, o, 65, f, 0, R, K, N) == S);
  EXPECT(G(NULL, 16, q, b, 16, sb, o, E, f, 0, R, K, N) == S && G(q, 16, NULL, b, 16, sb, o, E, f, 0, R, K, N) == S);
  EXPECT(G(q, 16, q, NULL, 16, sb, o, E, f, 0, R, K, N) == S && G(q, 16, q, b, 16, NULL, o, E, f, 0, R, K, N) == S);
  EXPECT(G(q, 16, q, b, 16, sb, NULL, E, f, 0, R, K, N) == S && G(q, 16, q, b, 16, sb, o, E, NULL, 0, R, K, N) == S);
  EXPECT(G(q, 16, q, b, 16, sb, o, E, f, 3, R, K, N) == U && G(q, 16, q, b, 16, sb, o, E, f, 0, 0, K, N) == S);
  EXPECT(G(q, 16, q, b, 16, sb, o, E, f, 0, R, 16, N) == S && G(q, 24, q, b, 16, sb, o, E, f, 0, R, K, N) == S);
  EXPECT(G(q, 16, q, b, 16, sb, (const uint32_t *)(q + 2), E, f, 0, R, K, N) == S);
  b[E - 1] = NULL;
  EXPECT(G(q, 16, q, b, 16, sb, o, E, f, 0, R, K, N) == S);
  b[E - 1] = q + 8;
  EXPECT(G(q, 16, q, b, 16, sb, o, E, f, 0, R, K, N) == S);
  b[E - 1] = q, sb[0] = NULL;
  EXPECT(G(q, 16, q, b, 16, sb, o, E, f, 0, R, K, N) == S);
  sb[0] = q + 2;
  EXPECT(G(q, 16, q, b, 16, sb, o, E, f, 0, R, K, N) == S);
  free(b), free(sb);
  void **dw = malloc(E * sizeof(*dw));
  if (!dw) abort();
  for (int e = 0; e < E; e++) dw[e] = q + 4096 * (E - e);
#define W(a, lda, sa, bq, ldb, sbq, off, e, out, yt, r, n, k) \
  grad(c, a, lda, sa, bq, ldb, sbq, off, e, out, (frx_dtype)(yt), r, n, k)
  EXPECT(W(q, 16, q, q, 16, q, o, 0, dw, 0, 32, N, K) == S && W(q, 16, q, q, 16, q, o, 65, dw, 0, 32, N, K) == S);
  EXPECT(W(q, 16, q, q, 16, q, NULL, E, dw, 0, 32, N, K) == S && W(q, 16, q, q, 16, q, o, E, NULL, 0, 32, N, K) == S);
  EXPECT(W(NULL, 16, q, q, 16, q, o, E, dw, 0, 32, N, K) == S && W(q, 16, NULL, q, 16, q, o, E, dw, 0, 32, N, K) == S);
  EXPECT(W(q, 16, q, NULL, 16, q, o, E, dw, 0, 32, N, K) == S && W(q, 16, q, q, 16, NULL, o, E, dw, 0, 32, N, K) == S);
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 0, 0, N, K) == S && W(q, 16, q, q, 16, q, o, E, dw, 0, 16, N, K) == S);
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 0, 64, N, K) == S && W(q, 24, q, q, 16, q, o, E, dw, 0, 32, N, K) == S);
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 2, 32, N, K) == U && W(q + 8, 16, q, q, 16, q, o, E, dw, 0, 32, N, K) == S);
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 0, 32, 0, K) == S && W(q, 16, q, q, 16, q, o, E, dw, 0, 32, N, 0) == S);
  EXPECT(W(q, 16, q, q, 16, q, (const uint32_t *)(q + 2), E, dw, 0, 32, N, K) == S);
  dw[1] = q + 1;
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 1, 32, N, K) == S);
  dw[1] = NULL;
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 0, 32, N, K) == S);
  dw[1] = dw[2];
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 0, 32, N, K) == S); /* two of one matrix */
  dw[1] = (char *)dw[2] + N * K * 4 - 4;
  EXPECT(W(q, 16, q, q, 16, q, o, E, dw, 0, 32, N, K) == S); /* one element of two */
  free(dw);
}

static void check_layer(frx_ctx *c, void *mem) {
  const frx_status S = FRX_ERR_SHAPE, U = FRX_ERR_UNSUPPORTED;
  enum { E = 3 };
  uint8_t *q = mem;
  float *f = mem;
  uint32_t *i = mem;
  const uint8_t **w[6];
  for (int k = 0; k < 6; k++) {
    w[k] = malloc(E * sizeof(*w[k]));
    if (!w[k]) abort();
    for (int e = 0; e < E; e++) w[k][e] = q;
  }
#define F(x, xt, r, rt, t, h, n, e, k, a, y, yt, idx, wt)                                                            \
  ffn(c, x, (frx_dtype)(xt), r, (frx_dtype)(rt), w[0], w[1], w[2], w[3], w[4], w[5], t, h, n, e, k, (frx_activation)(a), \
      y, (frx_dtype)(yt), idx, wt)
  EXPECT(F(NULL, 0, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == S && F(f, 0, f, 0, 1, 32, 32, E, 2, 0, NULL, 0, i, f) == S);
  EXPECT(F(f, 0, NULL, 0, 1, 32, 32, E, 2, 0, f, 0, NULL, f) == S && F(f, 0, NULL, 0, 1, 32, 32, E, 2, 0, f, 0, i, NULL) == S);
  EXPECT(F(f, 2, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == U && F(f, 0, f, 2, 1, 32, 32, E, 2, 0, f, 0, i, f) == U);
  EXPECT(F(f, 0, f, 0, 1, 32, 32, E, 2, 9, f, 0, i, f) == U && F(f, 0, f, 0, 1, 32, 32, E, 2, 0, f, 2, i, f) == U);
  EXPECT(F(f, 0, f, 0, 0, 32, 32, E, 2, 0, f, 0, i, f) == S && F(f, 0, f, 0, 65, 32, 32, E, 2, 0, f, 0, i, f) == U);
  EXPECT(F(f, 0, f, 0, 1, 0, 32, E, 2, 0, f, 0, i, f) == S && F(f, 0, f, 0, 1, 32, 0, E, 2, 0, f, 0, i, f) == S);
  EXPECT(F(f, 0, f, 0, 1, 48, 32, E, 2, 0, f, 0, i, f) == S && F(f, 0, f, 0, 1, 32, 48, E, 2, 0, f, 0, i, f) == S);
  EXPECT(F(f, 0, f, 0, 1, (1u << 23) + 32, 32, E, 2, 0, f, 0, i, f) == S);
  EXPECT(F(f, 0, f, 0, 1, 32, 0xFFFFFFE0u, E, 2, 0, f, 0, i, f) == S);
  EXPECT(F(f, 0, f, 0, 1, 32, 32, 0, 2, 0, f, 0, i, f) == S && F(f, 0, f, 0, 1, 32, 32, 65, 2, 0, f, 0, i, f) == S);
  EXPECT(F(f, 0, f, 0, 1, 32, 32, E, 0, 0, f, 0, i, f) == S && F(f, 0, f, 0, 1, 32, 32, E, E + 1, 0, f, 0, i, f) == S);
  EXPECT(F(f, 0, NULL, 0, 1, 32, 32, E, 65, 0, f, 0, i, f) == S);
  EXPECT(F(q + 2, 0, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == S && F(q + 1, 1, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == S);
  EXPECT(F(f, 0, q + 2, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == S && F(f, 0, f, 0, 1, 32, 32, E, 2, 0, q + 2, 0, i, f) == S);
  EXPECT(F(f, 0, f, 0, 1, 32, 32, E, 2, 0, f, 0, (uint32_t *)(q + 2), f) == S);
  EXPECT(F(f, 0, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, (float *)(q + 2)) == S);
  for (int k = 0; k < 6; k++) {
    const uint8_t **all = w[k];
    w[k] = NULL;
    EXPECT(F(f, 0, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == S);
    w[k] = all;
    w[k][E - 1] = NULL;
    EXPECT(F(f, 0, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == S);
    w[k][E - 1] = q + (k % 2 ? 2 : 8);
    EXPECT(F(f, 0, f, 0, 1, 32, 32, E, 2, 0, f, 0, i, f) == S);
    w[k][E - 1] = q;
  }
  for (int k = 0; k < 6; k++) free(w[k]);
}

/* Which calls allocate (zero codes under the smallest scale: every sum is 0). */
static void check_workspaces(frx_ctx *c, uint8_t *zeros, void *out) {
  size_t live = 1, retired = 1;
  uint32_t allocs = 1;
  const uint8_t *one[1] = {zeros};
  EXPECT(linear(c, zeros, 16, zeros, zeros, 16, zeros, out, FRX_F32, 40, 32, 8) == FRX_OK);
  EXPECT(act(c, zeros, FRX_F32, zeros, 16, zeros, out, FRX_F32, 16, 32, 8) == FRX_OK);
  EXPECT(grouped(c, zeros, 16, zeros, one, 16, one, (const uint32_t *)(void *)zeros, 1, out, FRX_F32, 8, 32, 8) == FRX_OK);
  EXPECT(frx_synchronize(c) == FRX_OK);
  EXPECT(frx_workspace_stats(c, &live, &retired, &allocs) == FRX_OK && live == 0 && allocs == 0);
  EXPECT(act(c, zeros, FRX_F32, zeros, 16, zeros, out, FRX_F32, 17, 32, 8) == FRX_OK);
  EXPECT(frx_workspace_stats(c, &live, &retired, &allocs) == FRX_OK && allocs == 1);
  EXPECT(act(c, zeros, FRX_BF16, zeros, 16, zeros, out, FRX_F32, 17, 32, 8) == FRX_OK);
  EXPECT(frx_workspace_stats(c, &live, &retired, &allocs) == FRX_OK && allocs == 1);
  EXPECT(ffn(c, zeros, FRX_F32, NULL, FRX_F32, one, one, one, one, one, one, 2, 32, 32, 1, 1, FRX_ACT_SILU, out, FRX_F32,
             (uint32_t *)(void *)zeros, (float *)(void *)zeros) == FRX_OK);
  EXPECT(frx_workspace_stats(c, &live, &retired, &allocs) == FRX_OK && allocs == 2 && retired == 0);
  EXPECT(frx_synchronize(c) == FRX_OK);
}

static void check_device(void) {
  frx_ctx *c = NULL;
  if (frx_create(0, &c) != FRX_OK || !c) {
    fprintf(stderr, "frx_create(0) failed\n");
    failures++;
    return;
  }
  /* twice 64 KB of device memory */
  uint8_t *zeros = calloc(65536, 1);
  uint32_t *mem = NULL, *out = NULL;
  float *scales[2] = {NULL, NULL};
  if (!zeros) abort();
  EXPECT(frx_upload_ternary(c, zeros, 64, 4096, NULL, 1.0f, &mem, &scales[0]) == FRX_OK);
  EXPECT(frx_upload_ternary(c, zeros, 64, 4096, NULL, 1.0f, &out, &scales[1]) == FRX_OK);
  free(zeros);
  if (mem && out) {
    check_products(c, mem);
    check_layer(c, mem);
    /* forced status: returned before any argument is read */
    const frx_status O = FRX_ERR_OOM;
    EXPECT(frx_force_status(c, O) == FRX_OK);
    EXPECT(quantize(c, NULL, FRX_F32, 0, 0, 0, FRX_FP4_ROWS, NULL, 0, NULL) == O);
    EXPECT(dequantize(c, NULL, 0, NULL, 0, 0, NULL, FRX_F32, 0) == O);
    EXPECT(linear(c, NULL, 0, NULL, NULL, 0, NULL, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(act(c, NULL, FRX_F32, NULL, 0, NULL, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(grouped(c, NULL, 0, NULL, NULL, 0, NULL, NULL, 0, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(grad(c, NULL, 0, NULL, NULL, 0, NULL, NULL, 0, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(ffn(c, NULL, FRX_F32, NULL, FRX_F32, NULL, NULL, NULL, NULL, NULL, NULL, 0, 0, 0, 0, 0, FRX_ACT_SILU, NULL,
               FRX_F32, NULL, NULL) == O);
    EXPECT(frx_force_status(c, FRX_OK) == FRX_OK);
    size_t live = 1, retired = 1;
    uint32_t allocs = 1;
    EXPECT(frx_workspace_stats(c, &live, &retired, &allocs) == FRX_OK);
    EXPECT(live == 0 && retired == 0 && allocs == 0); /* no refused call allocated */
    check_workspaces(c, (uint8_t *)mem, out);
    EXPECT(frx_free(c, mem) == FRX_OK && frx_free(c, scales[0]) == FRX_OK);
    EXPECT(frx_free(c, out) == FRX_OK && frx_free(c, scales[1]) == FRX_OK);
  }
  EXPECT(frx_synchronize(c) == FRX_OK);
  frx_destroy(c);
}

int main(int argc, char **argv) {
  const int device = argc > 1 && strcmp(argv[1], "--device") == 0;
  check_host();
  if (device) check_device();
  if (failures) {
    fprintf(stderr, "%d check(s) failed\n", failures);
    return 1;
  }
  printf("asan_fp4_check ok%s\n", device ? " (device validation)" : "");
  return 0;
}
