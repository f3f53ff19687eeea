// frx_fp8_ring.hpp — the 8-bit product for many tokens, software-pipelined.
//
// A tile of 32 * FM tokens x 256 weight rows on 8 waves of 16 * FM x 64, two to a
// SIMD, over two LDS stages (three at 128 tokens), one block of 128 columns
// each. Large tiles: what a compute unit reads per product halves from 128 x 128
// to 256 x 256, and so does the rate at which the L2's latency has to be
// covered. On the 8-bit pipe bound by issue: 4 multiply-adds beside each product,
// the DMA's and the operands' instructions (8192^3 in 256 x 256 tiles 374 us,
// without any DMA 306), and by power (fp8_plan). On the bf16 pipe the widening of
// the operands comes on top: a token fragment's 16 conversions for its 4 products in
// every wave (8192^3 in 192 x 256 tiles 931). Step t issues block t's products, and
// between them
//  - the multiply-adds of the token fragment before (the last one's of block
//    t - 1 behind the first products of block t), so that no product waits for
//    another's result;
//  - the operand reads one token fragment ahead; the weight operands of block
//    t + 1 replace block t's as the last token fragment uses them.
// Two barriers a step. Behind the first token fragment every wave has block t's
// weights in registers, so the DMA of a later block's weights (t + 2 with two
// stages) goes into their place. Before the last one block t + 1 has landed
// (each wave has waited for its own loads) and block t's tokens are read, so
// the later block's follow: each at least a step ahead of its use, spread over
// the products (8-bit pipe: in two bursts 2048 x 4096 x 11008 took 104 us, spread 88;
// in one 134).
#pragma once
#include "frx_fp8.hpp"

namespace frx {

// Waits for this wave's LDS reads, and for all but its last N loads.
template <int N>
__device__ __forceinline__ void wait_all_but() {
  static_assert(N < 16, "vmcnt's low bits");
  __builtin_amdgcn_s_waitcnt(N | (0x7 << 4));
}

// BR1: a scale per weight row, else per 128 of them. WIDE: the bf16 pipe; an
// operand is widened as it leaves LDS.
template <int FM_, bool E5M2, bool BR1, bool WIDE>
struct Fp8Ring {
  using Pipe = Fp8Pipe<WIDE>;
  static constexpr int FM = FM_, FN = 4, WM = 2, WN = 4, WAVES = WM * WN, NT = WAVES * 64;
  static constexpr int TM = FM * 16, TN = FN * 16, BM = WM * TM, BN = WN * TN;
  static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // 1 KB load instructions of a wave and stage
  static_assert(FM >= 4 && FM % 2 == 0, "loads split evenly; products alternate between two sets; loads between barriers");
  static constexpr int SIA = (BM + 63) / 64, SIB = BR1 ? BN / 64 : 1;  // scale load instructions
  static constexpr int SPW = (SIA + SIB + WAVES - 1) / WAVES;
  static constexpr int DATA = (BM + BN) * 32;  // dwords
  static constexpr int STAGE = DATA + SPW * WAVES * 64;
  // Stages: as many as fit, up to three.
  static constexpr int NS = 3 * STAGE * 4 <= 160 << 10 ? 3 : 2;
  static constexpr int LDS_BYTES = NS * STAGE * 4;
  static_assert(LDS_BYTES <= 160 << 10, "stages");
  // Whether a block's last multiply-adds wait for the next block's products (a
  // row's scales would have to be kept beside the next block's).
  static constexpr bool CARRY = !BR1;

  // Load instruction i of a wave covers 8 rows: a lane's offset in them (two,
  // as the swizzle of neighbouring groups of 8 rows differs) and, in the scalar
  // offset, the group's first row, clamped to the last group that has a valid
  // row. Rows past the valid ones in that group are past the buffer's end.
  struct Ctx {
    __amdgpu_buffer_rsrc_t ra, rb, rsa, rsb;
    uint32_t av[2], bv[2], sv[SPW];
    uint32_t lda8, ldb8, a_last, b_last;  // bytes of 8 rows; of the last valid group's first row
    int wave, last;
  };

  // One of the LA + LB + SPW loads of block kb (past the end the last one
  // again, into a stage that is not read).
  __device__ __forceinline__ static void load(int i, uint32_t *st, const Ctx &c, int kb) {
    kb = min(kb, c.last);
    const uint32_t k0 = 128u * (uint32_t)kb;
    if (i < LA) {
      const uint32_t row = min((uint32_t)(c.wave * LA + i) * c.lda8, c.a_last);
      lds_load16(c.ra, st + (c.wave * LA + i) * 256, c.av[i & 1], row + k0);
    } else if (i < LA + LB) {
      const int j = i - LA;
      const uint32_t row = min((uint32_t)(c.wave * LB + j) * c.ldb8, c.b_last);
      lds_load16(c.rb, st + BM * 32 + (c.wave * LB + j) * 256, c.bv[j & 1], row + k0);
    } else {
      const int j = i - LA - LB, s = c.wave * SPW + j;
      uint32_t *d = st + DATA + s * 64;
      if (s < SIA) lds_load4(c.rsa, d, c.sv[j], 4u * (uint32_t)kb);
      else lds_load4(c.rsb, d, c.sv[j], 4u * (uint32_t)kb);
    }
  }
  static constexpr int LOADS = LA + LB + SPW;
  // When a step issues them: the weights' with the products behind its first
  // barrier, EARLY of the tokens' with those behind its second one and the
  // late rest with the next step's first. A wave's burst of all of them
  // would fill the memory pipe's queue and block its products behind it.
  static constexpr int EARLY = LA < 2 ? LA : 2;
  __device__ static constexpr bool late(int i) { return i >= LA + LB || (i >= EARLY && i < LA); }

  __device__ static void run(uint32_t *lds, const Fp8Operands &o, f32x4 (&acc)[FN][FM]) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    Ctx c;
    c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = c.wave % WM, wn = c.wave / WM;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int ra = ((c.wave * LA + h) & 1) * 8 + (lane >> 3), rb = ((c.wave * LB + h) & 1) * 8 + (lane >> 3);
      c.av[h] = (uint32_t)(lane >> 3) * o.lda + 16 * ((lane & 7) ^ xswz(ra));
      c.bv[h] = (uint32_t)(lane >> 3) * o.ldb + 16 * ((lane & 7) ^ xswz(rb));
    }
    c.lda8 = 8 * o.lda;
    c.ldb8 = 8 * o.ldb;
    c.a_last = (uint32_t)((o.a_rows - 1) >> 3) * c.lda8;
    c.b_last = (uint32_t)((o.b_rows - 1) >> 3) * c.ldb8;
#pragma unroll
    for (int j = 0; j < SPW; j++) {
      const int s = c.wave * SPW + j;
      if (s < SIA) c.sv[j] = (uint32_t)min(s * 64 + lane, o.a_rows - 1) * o.sa_ld * 4;
      else if (BR1) c.sv[j] = (uint32_t)min((s - SIA) * 64 + lane, o.b_rows - 1) * o.sb_ld * 4;
      else c.sv[j] = (uint32_t)((o.b_first + min(lane * TN, o.b_rows - 1)) >> 7) * o.sb_ld * 4;  // lane w: wave column w's block
    }
    c.ra = buffer_rsrc(o.a, (uint32_t)(o.a_rows - 1) * o.lda + o.K);
    c.rb = buffer_rsrc(o.b, (uint32_t)(o.b_rows - 1) * o.ldb + o.K);
    const uint32_t kbs = (uint32_t)(o.K + 127) >> 7;
    c.rsa = buffer_rsrc(o.sa, ((uint32_t)(o.a_rows - 1) * o.sa_ld + kbs) * 4);
    c.rsb = buffer_rsrc(o.sb, ((uint32_t)(BR1 ? o.b_rows - 1 : (o.b_first + o.b_rows - 1) >> 7) * o.sb_ld + kbs) * 4);
#pragma unroll
    for (int fn = 0; fn < FN; fn++)
#pragma unroll
      for (int fm = 0; fm < FM; fm++) acc[fn][fm] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // dword offsets of this lane's operands in a stage: token fragment fm is
    // 16 rows (512 dwords) on, as is weight fragment fn
    const int lo = ((2 * g) ^ xswz(l16)) * 4, hi = ((2 * g + 1) ^ xswz(l16)) * 4;
    const int xo = (wm * TM + l16) * 32, wo = (BM + wn * TN + l16) * 32;
    const int so = DATA + wm * TM + l16;                                         // a token's scale
    const int bo = DATA + SIA * 64 + (BR1 ? wn * TN + 4 * g : wn);               // the weights'
    const auto op = [&](const uint32_t *st, int at) {
      const u32x4 a = *reinterpret_cast<const u32x4 *>(st + at + lo), b = *reinterpret_cast<const u32x4 *>(st + at + hi);
      return (i32x8){(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    };
    const auto add = [&](f32x4 &a, const f32x4 &p, float s, const f32x4 &sw) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (BR1) a[e] += p[e] * s * sw[e];
        else a[e] += p[e] * s;
      }
    };
    const int full = min(o.kb1, o.K >> 7);  // whole blocks; at most one more behind them
    if (o.kb0 < full) {
      c.last = full - 1;
#pragma unroll
      for (int i = 0; i < LOADS; i++) load(i, lds, c, o.kb0);
      if constexpr (NS == 3)
#pragma unroll
        for (int i = 0; i < LOADS; i++) load(i, lds + STAGE, c, o.kb0 + 1);
#pragma unroll
      for (int i = 0; i < LOADS; i++)
        if (!late(i)) load(i, lds + (NS - 1) * STAGE, c, o.kb0 + NS - 1);
      wait_vmcnt<(NS - 2) * LOADS + LB + EARLY>();
      barrier_nofence();
      typename Pipe::Op w[FN];
      i32x8 xc;  // the next token fragment
      f32x4 p[2][FN], sw[FN] = {};
      float sn, s[2] = {0.f, 0.f};
      Fp8Block sb;
#pragma unroll
      for (int fn = 0; fn < FN; fn++) {
        w[fn] = Pipe::template op<false>(op(lds, wo + fn * 512));
        p[1][fn] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (BR1) sw[fn] = *reinterpret_cast<const f32x4 *>(lds + bo + fn * 16);
      }
      if (!BR1) sb = Fp8Block(reinterpret_cast<const float *>(lds)[bo]);
      xc = op(lds, xo);
      sn = reinterpret_cast<const float *>(lds)[so];
      Fp8Factor xf = fp8_factor<WIDE, BR1>(sn, sb);
      int at = 0;  // dwords to the stage of block kb
      for (int kb = o.kb0; kb < full; kb++) {
        uint32_t *cur = lds + at;
        if (NS == 2) at ^= STAGE;
        else at = at == (NS - 1) * STAGE ? 0 : at + STAGE;
        uint32_t *nxt = lds + at;
        uint32_t *prv = nxt;  // the stage of block kb - 1 (and of kb - 1 + NS)
        if (NS == 3) prv = lds + (at == 2 * STAGE ? 0 : at + STAGE);
        float sbn = 0.f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int fm = 0; fm < FM; fm++) {
          const bool end = fm == FM - 1;
          if (fm == 0) {
#pragma unroll
            for (int i = 0; i < LOADS; i++)
              if (late(i)) load(i, prv, c, kb - 1 + NS);
          }
          if (fm == 1) {
            barrier_nofence();
            __builtin_amdgcn_sched_barrier(0);
          }
          if (end) {
            // in flight behind block kb + 1: whole blocks up to kb + NS, and of that one the weights
            wait_all_but<(NS - 2) * LOADS + LB>();
            barrier_nofence();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < EARLY; i++) load(i, cur, c, kb + NS);
          }
          // the weights' loads, a part to each fragment between the barriers
          constexpr int PER = (LB + FM - 3) / (FM - 2);
          if (fm >= 1 && !end) {
            const int first = (fm - 1) * PER;
#pragma unroll
            for (int i = first; i < first + PER && i < LB; i++) load(LA + i, cur, c, kb + NS);
          }
          const auto x = Pipe::template op<E5M2>(xc, xf.f);
          s[fm & 1] = xf.s;
          // the next fragment's operand
          const uint32_t *st = end ? nxt : cur;
          xc = op(st, xo + (fm + 1) % FM * 512);
          sn = reinterpret_cast<const float *>(st)[so + (fm + 1) % FM * 16];
          if (end && !BR1) sbn = reinterpret_cast<const float *>(nxt)[bo];
          i32x8 wr[FN];
          if (end && WIDE)
#pragma unroll
            for (int fn = 0; fn < FN; fn++) wr[fn] = op(nxt, wo + fn * 512);
#pragma unroll
          for (int fn = 0; fn < FN; fn++) {
            p[fm & 1][fn] = Pipe::template mul<E5M2>(w[fn], x);
            if (end) w[fn] = Pipe::template op<false>(WIDE ? wr[fn] : op(nxt, wo + fn * 512));
            if (CARRY || fm > 0) add(acc[fn][(fm + FM - 1) % FM], p[(fm + 1) & 1][fn], s[(fm + 1) & 1], sw[fn]);
          }
          if (end && !BR1) sb = Fp8Block(sbn);
          xf = fp8_factor<WIDE, BR1>(sn, sb);
          // a product; the operand reads behind the first; its multiply-adds
#pragma unroll
          for (int fn = 0; fn < FN; fn++) {
            __builtin_amdgcn_sched_group_barrier(0x008, WIDE ? 4 : 1, 0);
            if (fn == 0) {
              if (end && WIDE) __builtin_amdgcn_sched_group_barrier(0x100, 4 + 2 * FN, 0);
              else __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            } else if (end && !WIDE) {
              __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
            if (BR1) __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
            else __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (end && !CARRY) {
#pragma unroll
            for (int fn = 0; fn < FN; fn++) {
              add(acc[fn][FM - 1], p[fm & 1][fn], s[fm & 1], sw[fn]);
              sw[fn] = *reinterpret_cast<const f32x4 *>(nxt + bo + fn * 16);
            }
          }
        }
      }
      if (CARRY)
#pragma unroll
        for (int fn = 0; fn < FN; fn++) add(acc[fn][FM - 1], p[1][fn], s[1], sw[fn]);
      wait_vmcnt<0>();  // nothing is in flight into LDS any more
    }
    if (full < o.kb1) {  // the block that ends before its 128 columns, by itself
      __syncthreads();
      c.last = full;
#pragma unroll
      for (int i = 0; i < LOADS; i++) load(i, lds, c, full);
      wait_vmcnt<0>();
      __syncthreads();
      fp8_clear_tail(lds, BM + BN, full * 128, o.K, NT);
      __syncthreads();
      const float *sc = reinterpret_cast<const float *>(lds);
#pragma unroll
      for (int fm = 0; fm < FM; fm++) {
        const Fp8Factor xf = fp8_factor<WIDE, BR1>(sc[so + fm * 16], Fp8Block(BR1 ? 0.f : sc[bo]));
        const auto x = Pipe::template op<E5M2>(op(lds, xo + fm * 512), xf.f);
#pragma unroll
        for (int fn = 0; fn < FN; fn++) {
          const f32x4 sw = BR1 ? *reinterpret_cast<const f32x4 *>(lds + bo + fn * 16) : (f32x4){0.f, 0.f, 0.f, 0.f};
          add(acc[fn][fm], Pipe::template mul<E5M2>(Pipe::template op<false>(op(lds, wo + fn * 512)), x), xf.s, sw);
        }
      }
    }
  }

  template <typename YT>
  __device__ __forceinline__ static void store(const f32x4 (&acc)[FN][FM], YT *y, size_t ldy, int m_rows, int n_rows,
                                               bool vec) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    fp8_store<FN, FM>(acc, y, ldy, (wave % WM) * TM + (lane & 15), (wave / WM) * TN + 4 * (lane >> 4), m_rows, n_rows,
                      vec);
  }
};

}  // namespace frx
