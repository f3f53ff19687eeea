/* The 8-bit linears' and the expert sort's entry points as C declares them,
 * with the host code (frx_api.cpp) under AddressSanitizer and UBSan:
 *
 *  - Their signatures, and the room for sorted rows.
 *  - Every one with a null context returns FRX_ERR_DEVICE.
 *  - With "--device" (a GPU present) every argument check on a real context:
 *    null pointers, empty and oversized shapes, strides, alignments, types,
 *    experts, host arrays of exactly E entries on the heap, and the forced
 *    status. All are rejected before a launch; the pointers are device memory
 *    all the same.
 * Prints "asan_fp8_check ok" and exits 0 when every check passes. */
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
static frx_status (*const quantize)(frx_ctx *, const void *, frx_dtype, uint32_t, uint32_t, size_t, frx_fp8_blocks,
                                    frx_fp8, uint8_t *, size_t, float *) = frx_fp8_quantize;
static frx_status (*const sums)(frx_ctx *, frx_fp8_sums) = frx_set_fp8_sums;
static frx_status (*const linear)(frx_ctx *, const uint8_t *, size_t, frx_fp8, const float *, const uint8_t *, size_t,
                                  const float *, uint32_t, void *, frx_dtype, uint32_t, uint32_t,
                                  uint32_t) = frx_fp8_linear;
static frx_status (*const act)(frx_ctx *, const void *, frx_dtype, const uint8_t *, size_t, const float *, void *,
                               frx_dtype, uint32_t, uint32_t, uint32_t) = frx_fp8_linear_act;
static frx_status (*const grouped)(frx_ctx *, const uint8_t *, size_t, frx_fp8, const float *, const uint8_t *const *,
                                   size_t, const float *const *, const uint32_t *, uint32_t, void *, frx_dtype,
                                   uint32_t, uint32_t, uint32_t) = frx_fp8_linear_grouped;
static frx_status (*const grad)(frx_ctx *, const uint8_t *, size_t, frx_fp8, const float *, const uint8_t *, size_t,
                                const float *, const uint32_t *, uint32_t, void *const *, frx_dtype, uint32_t,
                                uint32_t, uint32_t) = frx_fp8_grad_weight_grouped;
static size_t (*const capacity)(uint32_t, uint32_t, uint32_t, uint32_t) = frx_moe_rows_capacity;
static frx_status (*const sort)(frx_ctx *, const uint32_t *, const frx_moe_rows *) = frx_moe_sort;
static frx_status (*const dispatch)(frx_ctx *, const void *, size_t, const frx_moe_rows *, void *) = frx_moe_dispatch;
static frx_status (*const combine)(frx_ctx *, const void *, frx_dtype, const frx_moe_rows *, const float *, void *,
                                   frx_dtype, uint32_t) = frx_moe_combine;
static frx_status (*const backward)(frx_ctx *, const void *, frx_dtype, const void *, frx_dtype, const frx_moe_rows *,
                                    const float *, void *, float *, uint32_t) = frx_moe_combine_backward;

static void check_host(void) {
  const frx_status D = FRX_ERR_DEVICE;
  EXPECT(capacity(0, 2, 8, 1) == 0);
  EXPECT(capacity(1, 1, 1, 1) == 1);
  EXPECT(capacity(10, 2, 4, 128) == 640);
  EXPECT(capacity(10, 2, 4, 0) == 0);
  EXPECT(capacity(0xFFFFFFFFu, 64, 64, 128) == ((size_t)0xFFFFFFFFu * 64 + 64 * 127 + 127) / 128 * 128);
  frx_moe_rows r;
  memset(&r, 0, sizeof(r));
  EXPECT(quantize(NULL, NULL, FRX_F32, 1, 1, 1, FRX_FP8_ROWS, FRX_FP8_E4M3, NULL, 16, NULL) == D);
  EXPECT(sums(NULL, FRX_FP8_SUMS_F32) == D);
  EXPECT(linear(NULL, NULL, 16, FRX_FP8_E4M3, NULL, NULL, 16, NULL, 128, NULL, FRX_F32, 1, 16, 1) == D);
  EXPECT(act(NULL, NULL, FRX_F32, NULL, 16, NULL, NULL, FRX_F32, 1, 16, 1) == D);
  EXPECT(grouped(NULL, NULL, 16, FRX_FP8_E4M3, NULL, NULL, 16, NULL, NULL, 1, NULL, FRX_F32, 1, 16, 1) == D);
  EXPECT(grad(NULL, NULL, 16, FRX_FP8_E4M3, NULL, NULL, 16, NULL, NULL, 1, NULL, FRX_F32, 16, 1, 1) == D);
  EXPECT(sort(NULL, NULL, &r) == D && sort(NULL, NULL, NULL) == D);
  EXPECT(dispatch(NULL, NULL, 4, &r, NULL) == D);
  EXPECT(combine(NULL, NULL, FRX_F32, &r, NULL, NULL, FRX_F32, 1) == D);
  EXPECT(backward(NULL, NULL, FRX_F32, NULL, FRX_F32, &r, NULL, NULL, NULL, 1) == D);
}

static void check_products(frx_ctx *c, void *mem) {
  const frx_status S = FRX_ERR_SHAPE, U = FRX_ERR_UNSUPPORTED;
  uint8_t *q = mem;
  float *f = mem;
  const uint32_t *o = mem;
  const size_t far = (size_t)1 << 23;
  /* the quantiser */
#define Q(x, xt, m, k, ldx, blocks, code, out, ldq, sc) \
  quantize(c, x, xt, m, k, ldx, (frx_fp8_blocks)(blocks), (frx_fp8)(code), out, ldq, sc)
  EXPECT(Q(NULL, FRX_F32, 2, 16, 16, 0, 0, q, 16, f) == S && Q(f, FRX_F32, 2, 16, 16, 0, 0, NULL, 16, f) == S);
  EXPECT(Q(f, FRX_F32, 2, 16, 16, 0, 0, q, 16, NULL) == S);
  EXPECT(Q(f, FRX_F32, 0, 16, 16, 0, 0, q, 16, f) == S && Q(f, FRX_F32, 2, 0, 16, 0, 0, q, 16, f) == S);
  EXPECT(Q(f, (frx_dtype)2, 2, 16, 16, 0, 0, q, 16, f) == U && Q(f, FRX_F32, 2, 16, 16, 4, 0, q, 16, f) == U);
  EXPECT(Q(f, FRX_F32, 2, 16, 16, 0, 2, q, 16, f) == U && Q(f, FRX_F32, 2, 16, 16, 0, 9, q, 16, f) == U);
  EXPECT(Q(f, FRX_F32, 2, 16, 15, 0, 0, q, 16, f) == S && Q(f, FRX_F32, 2, 16, 16, 0, 0, q, 24, f) == S);
  EXPECT(Q(f, FRX_F32, 2, 17, 17, 0, 0, q, 16, f) == S && Q(f, FRX_F32, 17, 2, 2, 1, 0, q, 16, f) == S);
  EXPECT(Q(f, FRX_F32, 17, 2, 2, 3, 0, q, 16, f) == S);
  EXPECT(Q((char *)mem + 2, FRX_F32, 2, 16, 16, 0, 0, q, 16, f) == S);
  EXPECT(Q((char *)mem + 1, FRX_BF16, 2, 16, 16, 0, 0, q, 16, f) == S);
  EXPECT(Q(f, FRX_F32, 2, 16, 16, 0, 0, q + 8, 16, f) == S);
  EXPECT(Q(f, FRX_F32, 2, 16, 16, 0, 0, q, 16, (float *)(q + 2)) == S);
  EXPECT(Q(f, FRX_F32, 0xFFFFFFFFu, 16, 16, 0, 0, q, 16, f) == S);
  EXPECT(Q(f, FRX_F32, 1u << 30, 128, 128, 0, 0, q, 128, f) == S);
  EXPECT(Q(f, FRX_F32, 1u << 20, 1u << 20, 1u << 20, 2, 0, q, 1u << 20, f) == S);
  EXPECT(strlen(frx_last_error(c)) > 0);
  /* one product */
#define L(a, lda, at, sa, b, ldb, sb, br, y, yt, m, k, n) \
  linear(c, a, lda, (frx_fp8)(at), sa, b, ldb, sb, br, y, (frx_dtype)(yt), m, k, n)
  EXPECT(L(NULL, 16, 0, f, q, 16, f, 128, f, 0, 1, 16, 1) == S && L(q, 16, 0, NULL, q, 16, f, 128, f, 0, 1, 16, 1) == S);
  EXPECT(L(q, 16, 0, f, NULL, 16, f, 128, f, 0, 1, 16, 1) == S && L(q, 16, 0, f, q, 16, NULL, 128, f, 0, 1, 16, 1) == S);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, NULL, 0, 1, 16, 1) == S && L(q, 16, 2, f, q, 16, f, 128, f, 0, 1, 16, 1) == U);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, f, 2, 1, 16, 1) == U && L(q, 16, 0, f, q, 16, f, 64, f, 0, 1, 16, 1) == U);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, f, 0, 0, 16, 1) == S && L(q, 16, 0, f, q, 16, f, 128, f, 0, 1, 0, 1) == S);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, f, 0, 1, 16, 0) == S && L(q, 32, 0, f, q, 32, f, 128, f, 0, 1, 24, 1) == S);
  EXPECT(L(q, 24, 0, f, q, 32, f, 128, f, 0, 1, 16, 1) == S && L(q, 32, 0, f, q, 24, f, 128, f, 0, 1, 16, 1) == S);
  EXPECT(L(q, 16, 0, f, q, 32, f, 128, f, 0, 1, 32, 1) == S && L(q, 32, 0, f, q, 16, f, 128, f, 0, 1, 32, 1) == S);
  EXPECT(L(q, far + 16, 0, f, q, 16, f, 128, f, 0, 1, 16, 1) == S && L(q, 16, 0, f, q, far + 16, f, 128, f, 0, 1, 16, 1) == S);
  EXPECT(L(q + 8, 16, 0, f, q, 16, f, 128, f, 0, 1, 16, 1) == S && L(q, 16, 0, f, q + 8, 16, f, 128, f, 0, 1, 16, 1) == S);
  EXPECT(L(q, 16, 0, (float *)(q + 2), q, 16, f, 128, f, 0, 1, 16, 1) == S);
  EXPECT(L(q, 16, 0, f, q, 16, (float *)(q + 2), 128, f, 0, 1, 16, 1) == S);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, q + 2, 0, 1, 16, 1) == S && L(q, 16, 0, f, q, 16, f, 128, q + 1, 1, 1, 16, 1) == S);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, f, 0, 0xFFFFFFFFu, 16, 1) == S);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, f, 0, 1, 16, 0xFFFFFFFFu) == S);
  EXPECT(L(q, 16, 0, f, q, 16, f, 128, f, 0, 1u << 20, 16, 1u << 20) == S);
  /* with the activations quantised inside */
#define A(x, xt, b, ldb, sb, y, yt, m, k, n) act(c, x, (frx_dtype)(xt), b, ldb, sb, y, (frx_dtype)(yt), m, k, n)
  EXPECT(A(NULL, 0, q, 16, f, f, 0, 1, 16, 1) == S && A(f, 2, q, 16, f, f, 0, 1, 16, 1) == U);
  EXPECT(A(q + 2, 0, q, 16, f, f, 0, 1, 16, 1) == S && A(q + 1, 1, q, 16, f, f, 0, 1, 16, 1) == S);
  EXPECT(A(f, 0, NULL, 16, f, f, 0, 1, 16, 1) == S && A(f, 0, q, 16, NULL, f, 0, 1, 16, 1) == S);
  EXPECT(A(f, 0, q, 16, f, NULL, 0, 1, 16, 1) == S && A(f, 0, q, 16, f, f, 2, 1, 16, 1) == U);
  EXPECT(A(f, 0, q, 32, f, f, 0, 1, 24, 1) == S && A(f, 0, q, 24, f, f, 0, 1, 16, 1) == S);
  EXPECT(A(f, 0, q, 16, f, f, 0, 0, 16, 1) == S && A(f, 0, q, 16, f, f, 0, 1, 16, 0) == S);
  EXPECT(A(f, 0, q, 2 * far, f, f, 0, 1, 2 * (uint32_t)far, 1) == S);
  /* experts: host arrays of exactly E entries */
  enum { E = 3, N = 4, K = 16, R = 16 };
  const uint8_t **b = malloc(E * sizeof(*b));
  const float **sb = malloc(E * sizeof(*sb));
  void **dw = malloc(E * sizeof(*dw));
  if (!b || !sb || !dw) abort();
  for (int e = 0; e < E; e++) b[e] = q, sb[e] = f, dw[e] = q + 4096 * (E - e);
#define G(a, lda, at, sa, bs, ldb, sbs, off, e, y, yt, r, k, n) \
  grouped(c, a, lda, (frx_fp8)(at), sa, bs, ldb, sbs, off, e, y, (frx_dtype)(yt), r, k, n)
  EXPECT(G(q, 16, 0, f, b, 16, sb, o, 0, f, 0, R, K, N) == S && G(q, 16, 0, f, b, 16, sb, o, 65, f, 0, R, K, N) == S);
  EXPECT(G(NULL, 16, 0, f, b, 16, sb, o, E, f, 0, R, K, N) == S && G(q, 16, 0, NULL, b, 16, sb, o, E, f, 0, R, K, N) == S);
  EXPECT(G(q, 16, 0, f, NULL, 16, sb, o, E, f, 0, R, K, N) == S && G(q, 16, 0, f, b, 16, NULL, o, E, f, 0, R, K, N) == S);
  EXPECT(G(q, 16, 0, f, b, 16, sb, NULL, E, f, 0, R, K, N) == S && G(q, 16, 0, f, b, 16, sb, o, E, NULL, 0, R, K, N) == S);
  EXPECT(G(q, 16, 3, f, b, 16, sb, o, E, f, 0, R, K, N) == U && G(q, 16, 0, f, b, 16, sb, o, E, f, 3, R, K, N) == U);
  EXPECT(G(q, 16, 0, f, b, 16, sb, o, E, f, 0, 0, K, N) == S && G(q, 16, 0, f, b, 16, sb, o, E, f, 0, R, 8, N) == S);
  EXPECT(G(q, 16, 0, f, b, 16, sb, (const uint32_t *)(q + 2), E, f, 0, R, K, N) == S);
  b[E - 1] = NULL;
  EXPECT(G(q, 16, 0, f, b, 16, sb, o, E, f, 0, R, K, N) == S);
  b[E - 1] = q + 8;
  EXPECT(G(q, 16, 0, f, b, 16, sb, o, E, f, 0, R, K, N) == S);
  b[E - 1] = q, sb[0] = NULL;
  EXPECT(G(q, 16, 0, f, b, 16, sb, o, E, f, 0, R, K, N) == S);
#define W(a, lda, at, sa, bq, ldb, sbq, off, e, out, yt, r, n, k) \
  grad(c, a, lda, (frx_fp8)(at), sa, bq, ldb, sbq, off, e, out, (frx_dtype)(yt), r, n, k)
  EXPECT(W(q, 16, 1, f, q, 16, f, o, 0, dw, 0, R, N, K) == S && W(q, 16, 1, f, q, 16, f, o, 65, dw, 0, R, N, K) == S);
  EXPECT(W(q, 16, 1, f, q, 16, f, NULL, E, dw, 0, R, N, K) == S && W(q, 16, 1, f, q, 16, f, o, E, NULL, 0, R, N, K) == S);
  EXPECT(W(NULL, 16, 1, f, q, 16, f, o, E, dw, 0, R, N, K) == S && W(q, 16, 1, f, NULL, 16, f, o, E, dw, 0, R, N, K) == S);
  EXPECT(W(q, 32, 1, f, q, 32, f, o, E, dw, 0, 24, N, K) == S && W(q, 16, 1, f, q, 16, f, o, E, dw, 2, R, N, K) == U);
  EXPECT(W(q, 16, 1, f, q, 16, f, (const uint32_t *)(q + 2), E, dw, 0, R, N, K) == S);
  dw[1] = q + 1;
  EXPECT(W(q, 16, 1, f, q, 16, f, o, E, dw, 1, R, N, K) == S);
  dw[1] = NULL;
  EXPECT(W(q, 16, 1, f, q, 16, f, o, E, dw, 0, R, N, K) == S);
  dw[1] = dw[2];
  EXPECT(W(q, 16, 1, f, q, 16, f, o, E, dw, 0, R, N, K) == S); /* two of one matrix */
  dw[1] = (char *)dw[2] + N * K * 4 - 4;
  EXPECT(W(q, 16, 1, f, q, 16, f, o, E, dw, 0, R, N, K) == S); /* one element of two */
  free(b), free(sb), free(dw);
  EXPECT(sums(c, (frx_fp8_sums)2) == U && sums(c, (frx_fp8_sums)9) == U);
  EXPECT(sums(c, FRX_FP8_SUMS_PIPE) == FRX_OK && sums(c, FRX_FP8_SUMS_F32) == FRX_OK);
}

static void check_routes(frx_ctx *c, void *mem) {
  const frx_status S = FRX_ERR_SHAPE, U = FRX_ERR_UNSUPPORTED;
  uint32_t *i = mem;
  float *f = mem;
  char *p = mem;
  const frx_moe_rows good = {4, 2, 8, 1, 8, i, i, i};
  EXPECT(sort(c, NULL, &good) == S && sort(c, i, NULL) == S && sort(c, (uint32_t *)(p + 2), &good) == S);
#define BAD(field, value)                                                  \
  do {                                                                     \
    frx_moe_rows r = good;                                                 \
    r.field = value;                                                       \
    EXPECT(sort(c, i, &r) == S);                                           \
    EXPECT(dispatch(c, p, 4, &r, p) == S);                                 \
    EXPECT(combine(c, f, FRX_F32, &r, f, f, FRX_F32, 4) == S);             \
    EXPECT(backward(c, f, FRX_F32, f, FRX_F32, &r, f, f, f, 4) == S);      \
  } while (0)
  BAD(T, 0);
  BAD(T, 5);           /* more rows than R */
  BAD(T, 0xFFFFFFFFu);
  BAD(top_k, 0);
  BAD(top_k, 65);
  BAD(E, 0);
  BAD(E, 65);
  BAD(align, 0);
  BAD(align, 3);
  BAD(align, 256);
  BAD(align, 128);     /* needs more rows */
  BAD(R, 7);
  BAD(R, 1u << 24);
  BAD(offsets, NULL);
  BAD(row_of, NULL);
  BAD(slot_of, NULL);
  BAD(offsets, (uint32_t *)(p + 2));
  BAD(row_of, (uint32_t *)(p + 1));
  BAD(slot_of, (uint32_t *)(p + 3));
  EXPECT(dispatch(c, NULL, 4, &good, p) == S && dispatch(c, p, 4, &good, NULL) == S);
  EXPECT(dispatch(c, p, 0, &good, p) == S && dispatch(c, p, 6, &good, p) == S);
  EXPECT(dispatch(c, p, ((size_t)1 << 30) + 4, &good, p) == S);
  EXPECT(dispatch(c, p + 2, 4, &good, p) == S && dispatch(c, p, 4, &good, p + 1) == S);
  EXPECT(combine(c, NULL, FRX_F32, &good, f, f, FRX_F32, 4) == S && combine(c, f, FRX_F32, &good, f, NULL, FRX_F32, 4) == S);
  EXPECT(combine(c, f, (frx_dtype)2, &good, f, f, FRX_F32, 4) == U && combine(c, f, FRX_F32, &good, f, f, (frx_dtype)2, 4) == U);
  EXPECT(combine(c, f, FRX_F32, &good, f, f, FRX_F32, 0) == S && combine(c, f, FRX_F32, &good, f, f, FRX_F32, 65535u * 256 + 1) == S);
  EXPECT(combine(c, p + 2, FRX_F32, &good, f, f, FRX_F32, 4) == S && combine(c, f, FRX_F32, &good, f, p + 1, FRX_BF16, 4) == S);
  EXPECT(combine(c, f, FRX_F32, &good, (float *)(p + 2), f, FRX_F32, 4) == S);
  EXPECT(backward(c, NULL, FRX_F32, f, FRX_F32, &good, f, f, f, 4) == S && backward(c, f, FRX_F32, f, FRX_F32, &good, f, NULL, f, 4) == S);
  EXPECT(backward(c, f, FRX_F32, NULL, FRX_F32, &good, f, f, f, 4) == S && backward(c, f, FRX_F32, f, FRX_F32, &good, f, f, NULL, 4) == S);
  EXPECT(backward(c, f, (frx_dtype)2, f, FRX_F32, &good, f, f, f, 4) == U && backward(c, f, FRX_F32, f, (frx_dtype)2, &good, f, f, f, 4) == U);
  EXPECT(backward(c, f, FRX_F32, f, FRX_F32, &good, f, f, f, 0) == S);
  EXPECT(backward(c, p + 2, FRX_F32, f, FRX_F32, &good, f, f, f, 4) == S && backward(c, f, FRX_F32, p + 2, FRX_F32, &good, f, f, f, 4) == S);
  EXPECT(backward(c, f, FRX_F32, f, FRX_F32, &good, f, p + 2, f, 4) == S);
  EXPECT(backward(c, f, FRX_F32, f, FRX_F32, &good, f, f, (float *)(p + 2), 4) == S);
  EXPECT(backward(c, f, FRX_F32, f, FRX_F32, &good, (float *)(p + 2), f, f, 4) == S);
}

static void check_device(void) {
  frx_ctx *c = NULL;
  if (frx_create(0, &c) != FRX_OK || !c) {
    fprintf(stderr, "frx_create(0) failed\n");
    failures++;
    return;
  }
  /* 64 KB of device memory */
  uint8_t *zeros = calloc(65536, 1);
  uint32_t *mem = NULL;
  float *scales = NULL;
  if (!zeros) abort();
  EXPECT(frx_upload_ternary(c, zeros, 64, 4096, NULL, 1.0f, &mem, &scales) == FRX_OK);
  free(zeros);
  if (mem) {
    check_products(c, mem);
    check_routes(c, mem);
    /* forced status: returned before any argument is read */
    const frx_status O = FRX_ERR_OOM;
    EXPECT(frx_force_status(c, O) == FRX_OK);
    EXPECT(quantize(c, NULL, FRX_F32, 0, 0, 0, FRX_FP8_ROWS, FRX_FP8_E4M3, NULL, 0, NULL) == O);
    EXPECT(linear(c, NULL, 0, FRX_FP8_E4M3, NULL, NULL, 0, NULL, 0, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(act(c, NULL, FRX_F32, NULL, 0, NULL, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(grouped(c, NULL, 0, FRX_FP8_E4M3, NULL, NULL, 0, NULL, NULL, 0, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(grad(c, NULL, 0, FRX_FP8_E4M3, NULL, NULL, 0, NULL, NULL, 0, NULL, FRX_F32, 0, 0, 0) == O);
    EXPECT(sort(c, NULL, NULL) == O && dispatch(c, NULL, 0, NULL, NULL) == O);
    EXPECT(combine(c, NULL, FRX_F32, NULL, NULL, NULL, FRX_F32, 0) == O);
    EXPECT(backward(c, NULL, FRX_F32, NULL, FRX_F32, NULL, NULL, NULL, NULL, 0) == O);
    EXPECT(frx_force_status(c, FRX_OK) == FRX_OK);
    size_t live = 1, retired = 1;
    uint32_t allocs = 1;
    EXPECT(frx_workspace_stats(c, &live, &retired, &allocs) == FRX_OK);
    EXPECT(live == 0 && retired == 0); /* no refused call allocated */
    EXPECT(frx_free(c, mem) == FRX_OK && frx_free(c, scales) == FRX_OK);
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
  printf("asan_fp8_check ok%s\n", device ? " (device validation)" : "");
  return 0;
}
