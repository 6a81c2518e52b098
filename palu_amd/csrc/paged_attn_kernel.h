// Decode attention of many sequences over the pages of a 4-bit latent cache: one new token of each of B sequences.
//
//   x_l     = (c_l - z_l) s_l                           the key latent of position l (codes c, an fp16 pair (scale s, zero z) a row)
//   score_l = sm_scale <R(pos) q, R(l) (x_l B_h)>       B_h [Rk, 128]: the head's key reconstruction, R(l) the rotation by l
//   ctx     = sum_l softmax(score)_l (v_l - zv_l) sv_l  the head's context in latent space
//
// The rotation of the query is moved to the keys (<R(p) q, R(l) k> = <q, R(l - p) k>), and the query is folded into B:
//   Fc[r, i] = q_i B[r, i] + q_{i+64} B[r, i+64]        Fs[r, i] = q_{i+64} B[r, i] - q_i B[r, i+64]
//   score_l  = s_l sum_i cos((l - p) w_i) Yc_i + sin((l - p) w_i) Ys_i,     Y = F^T (c_l - z_l)
// so no key is ever written down: Y is a matrix product (512 columns for four heads), the rotation a dot product in registers.
//
// Work: 2 Rk 512 + 2 Rv 4 flops a position and group of four heads against Rk / 2 + Rv / 2 + 8 bytes -- 500 flops a byte, so the
// matrix pipe and the vector units bound it, not the memory.  Split:
//   * A workgroup (8 waves) takes a range of tiles (128 positions; 64 where Rk > 128) of one (sequence, four heads of one latent
//     group: two where Rk > 128, whose fragments fill the registers).  The tiles of the whole batch are one line, cut into gridDim.x equal pieces, so ragged batches need no plan from the
//     host and replay in a graph; a piece that covers a sequence's end goes on with the next.  Pieces of one sequence are joined by
//     a second kernel.
//   * Scores: wave w owns the RoPE pairs 8 w .. 8 w + 7 of all heads.  Its part of F stays in registers (4 heads x 16 columns x Rk:
//     64 VGPRs at Rk = 128) as the A operand of v_mfma_f32_32x32x16_f16, two heads an instruction; a tile's codes are turned into
//     fp16 once, by all eight waves, and shared through LDS as the B operand.  A lane then holds 4 pairs of ONE position for two
//     heads, and the cos / sin of those 4 pairs, advanced from block to block by a rotation (exact again every 32 tiles), serve
//     all heads.  The eight waves' partial scores meet in LDS.
//   * Softmax and values: wave w owns an eighth of a tile's positions, with its own running maximum and sums; the eight are joined
//     at the end of the range.  A lane holds eight columns of one row, and v_mfma_f32_4x4x4_16b_f16 (16 independent blocks of
//     4 heads x 4 positions x 4 columns) wastes no row on the four heads a group has.
//   * The values of tile t - 1 run in the same barrier interval as the scores of tile t, in front of them in waves 4 .. 7 and behind
//     them in waves 0 .. 3: the two waves of a SIMD keep the matrix pipe and the vector unit busy at the same time.
#pragma once
#include "palu_common.h"

namespace {

constexpr int PA_THREADS = 512;
constexpr int PA_FIX = 3;                // cost of starting and ending a piece, in tiles (measured: 6 us against 2 us a tile)
constexpr int PA_SLAB = 2048;            // floats of a (wave, subset) slab times subsets: [4 heads][512 / S columns] of the epilogue

struct PagedAttnParams {
  const h16* q;       int64_t sq_b, sq_h;
  const h16* bfrag;                      // palu_paged_prepare_b's layout
  const unsigned* kc; const unsigned* km;
  const unsigned* vc; const unsigned* vm;
  const int* table;   int64_t st_b;
  const int* lens;
  const int* qpos;                       // null: q is rotated already
  const float* inv_freq;
  h16* ctx;
  float* part;                           // partial results: [slots][4][2] (maximum, sum), then [slots][4][Rv]
  int slots;
  int B, H, G, gs, VG;                   // gs = H / G heads of a latent group, dealt into VG sets of `heads` (2 or 4)
  int max_pages, log_p, n_pages, Rk, Rv;
  int heads;
  int tile;                              // positions of a tile
  int min_chunk;                         // tiles a workgroup takes at least
  int direct;                            // one workgroup per (sequence, heads): no partial results, no second kernel
  float scale;                           // sm_scale log2(e)
};

// A sequence's rows, and whether the table has room for them (a length beyond it poisons the sequence with NaN).
static __device__ __forceinline__ int pa_rows(const PagedAttnParams& p, int b) {
  return min(max(p.lens[b], 0), p.max_pages << p.log_p);
}
static __device__ __forceinline__ bool pa_bad_len(const PagedAttnParams& p, int b) { return p.lens[b] > (p.max_pages << p.log_p); }
static __device__ __forceinline__ int pa_tiles(const PagedAttnParams& p, int b) { return (pa_rows(p, b) + p.tile - 1) / p.tile; }

// The line of all work: sequences in order, for each its G VG sets of heads in order, for each a fixed part (the fold of the query and
// the join of the waves, PA_FIX tiles' worth) and its tiles.  The line is cut into gridDim.x equal pieces.
struct PaLine {
  int total;                             // length of the line
  int front;                             // of the sequences in front of sequence b
};
static __device__ __forceinline__ int pa_cost(const PagedAttnParams& p, int b) {
  const int n = pa_tiles(p, b);
  return n ? (n + PA_FIX) * p.G * p.VG : 0;
}
static __device__ __forceinline__ int wave_scan(int v, int lane) {            // inclusive sum over the wave
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  return v;
}
static __device__ __forceinline__ PaLine pa_line(const PagedAttnParams& p, int lane, int b) {
  int total = 0, front = 0;
  for (int i = lane; i < p.B; i += 64) {
    const int c = pa_cost(p, i);
    total += c;
    if (i < b) front += c;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    total += __shfl_xor(total, o, 64);
    front += __shfl_xor(front, o, 64);
  }
  return {total, front};
}
static __device__ __forceinline__ int pa_chunk(const PagedAttnParams& p, int total, int W) {
  return max((total + W - 1) / W, p.min_chunk + PA_FIX);
}

// maximum over the 16 lanes of a DPP row
static __device__ __forceinline__ float row_max16(float v) {
#define PA_ROR(N) v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, false)))
  PA_ROR(1); PA_ROR(2); PA_ROR(4); PA_ROR(8);
#undef PA_ROR
  return v;
}
static __device__ __forceinline__ float row_sum16(float v) {
#define PA_ROR(N) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, false))
  PA_ROR(1); PA_ROR(2); PA_ROR(4); PA_ROR(8);
#undef PA_ROR
  return v;
}
static __device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

template <int NKS>
struct PaLds {
  static constexpr int TILE = NKS <= 8 ? 128 : 64;
  static constexpr int XS = NKS * 32 + 16;                 // bytes of a position's row: 16 more, so that 8 lanes reading 16 bytes of 8 rows meet 8 bank groups
  static constexpr int RED = 2 * TILE * XS;                // float [2][8 waves][4 heads][TILE]
  static constexpr int WGT = RED + 2 * 8 * 4 * TILE * 4;   // h16 [8 waves]: weights [4 heads][16], zeros [16]
  static constexpr int STEP = WGT + 8 * 80 * 2;            // f32x4 [8 waves][2 halves][2]: cos / sin of a 32-position step
  static constexpr int LOOP = STEP + 8 * 64;
  static constexpr int STAT = 8 * PA_SLAB * 4;             // (epilogue, over the loop's) float [8 waves][4 heads][4], sums [4], maxima [4]
  static constexpr int BYTES = LOOP > STAT + 576 ? LOOP : STAT + 576;
};

// NKS: 16-column blocks of the (padded) key rank.  S: rows of values a wave holds side by side (Rv <= 512 / S).  NH: heads computed.
template <int NKS, int S, int NH>
__global__ __launch_bounds__(PA_THREADS, 2) void paged_attn_kernel(PagedAttnParams p) {
  using L = PaLds<NKS>;
  constexpr int TILE = L::TILE;
  constexpr int ROWS = TILE / 8;                           // positions of a tile that a wave owns
  constexpr int NB = TILE / 32;                            // 32-position blocks
  constexpr int MB = NH / 2;                               // matrix blocks of two heads
  constexpr int KL = 64 / ROWS;                            // lanes of a key row
  constexpr int UL = 2 * NKS / KL;                         // words of codes such a lane turns into fp16
  constexpr int ST = ROWS / (4 * S);                       // steps of 4 positions a block takes through a wave's rows
  static_assert(ST >= 1 && UL * KL == 2 * NKS, "a wave's rows");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hi = lane >> 5;
  const int GV = p.G * p.VG;
  float* const red = reinterpret_cast<float*>(smem + L::RED);
  h16* const wgt = reinterpret_cast<h16*>(smem + L::WGT) + w * 80;
  const f32x4* const step = reinterpret_cast<const f32x4*>(smem + L::STEP) + w * 4 + hi * 2;

  // ---- this workgroup's piece of the line
  int at = 0, end = 0;
  int b = 0;
  int base = 0;                                            // where sequence b begins on the line
  if (p.direct) {
    b = blockIdx.x / GV;
  } else {
    int c = 0, incl = 0, total = 0;
    if (p.B <= 64) {                                       // (one load of the lengths serves the sum and the search)
      c = lane < p.B ? pa_cost(p, lane) : 0;
      incl = wave_scan(c, lane);
      total = __shfl(incl, 63, 64);
    } else {
      total = pa_line(p, lane, -1).total;
    }
    const int chunk = pa_chunk(p, total, gridDim.x);
    const int64_t start = (int64_t)blockIdx.x * chunk;
    if (start >= total) return;                            // behind the line's end
    at = (int)start;
    end = (int)min(start + chunk, (int64_t)total);
    for (int i0 = 0;; i0 += 64) {                          // the sequence that holds `at`
      if (p.B > 64) {
        c = i0 + lane < p.B ? pa_cost(p, i0 + lane) : 0;
        incl = wave_scan(c, lane);
      }
      const unsigned long long past = __ballot(base + incl > at);
      if (past) {
        const int f = __ffsll((unsigned long long)past) - 1;
        b = i0 + f;
        base += __shfl(incl - c, f, 64);
        break;
      }
      base += __shfl(incl, 63, 64);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    base = __builtin_amdgcn_readfirstlane(base);
    at = __builtin_amdgcn_readfirstlane(at);
    end = __builtin_amdgcn_readfirstlane(end);
  }

  while (b < p.B) {
    const int nt = __builtin_amdgcn_readfirstlane(pa_tiles(p, b));
    if (nt == 0) {
      if (p.direct) break;
      ++b;
      continue;
    }
    int gv, t0, t1;
    if (p.direct) {
      gv = blockIdx.x - b * GV;
      t0 = 0;
      t1 = nt;
    } else {
      const int rel = at - base;                           // into sequence b
      gv = rel / (nt + PA_FIX);
      const int into = rel - gv * (nt + PA_FIX) - PA_FIX;  // tiles of this set of heads in front of `at` (negative: in its fixed part)
      t0 = max(into, 0);
      t1 = min(nt, into + (end - at));
      at += nt - into;                                     // where the next set begins
      if (t1 <= t0) break;                                 // (the piece ends inside the fixed part: its tiles are the next piece's)
    }
    const int g = gv / p.VG, vg = gv - g * p.VG;
    const int h0 = g * p.gs + NH * vg, nh = min(NH, p.gs - NH * vg);
    const int rows = __builtin_amdgcn_readfirstlane(pa_rows(p, b));
    const int qp = p.qpos ? p.qpos[b] : 0;
    const int* const table = p.table + (int64_t)b * p.st_b;

    // Pages of this wave's positions (ROWS of a tile, never across a page's end), of 64 tiles at once: lane i has tile tb + i's, so
    // that no tile waits for the table.  None: 0 (a page that exists; the rows are masked); outside the pool: -1.
    int pages = 0, tb = t0;
    auto load_pages = [&]() {
      const int64_t l = (int64_t)(tb + lane) * TILE + ROWS * w;
      pages = 0;
      if (tb + lane < t1 && l < rows) {
        pages = table[l >> p.log_p];
        if (pages >= p.n_pages) pages = -1;
      }
    };
    auto page_of = [&](int t, bool& bad) {                 // (t never falls back by a whole load)
      if (t - tb == 64) {
        tb = t;
        load_pages();
      }
      const int pg = __builtin_amdgcn_readlane(pages, t - tb);
      bad = pg < 0;
      return bad ? 0 : pg;
    };
    load_pages();
    auto slot_of = [&](int t, int pg) {                    // first row of those in the pool
      return (((int64_t)pg * p.G + g) << p.log_p) + ((t * TILE + ROWS * w) & ((1 << p.log_p) - 1));
    };

    // ---- loads of a tile: key codes (KL lanes a row) and their pairs; value codes (a lane 8 columns of ST x 4 rows) and the pairs
    unsigned kreg[UL], kmeta;
    const int krow = lane / KL, kpart = lane % KL;
    const int kw = p.Rk >> 3, vw = p.Rv >> 3;
    const unsigned klane = krow * kw + kpart * UL;
    auto load_k = [&](int64_t slot) {
      const unsigned* src = p.kc + slot * kw + klane;
      if (kw == KL * UL) {
#pragma unroll
        for (int i = 0; i < UL; ++i) kreg[i] = src[i];
      } else {
#pragma unroll
        for (int i = 0; i < UL; ++i) kreg[i] = kpart * UL + i < kw ? src[i] : 0u;
      }
      kmeta = (p.km + slot)[(unsigned)krow];
    };
    unsigned vreg[ST][4], smk, smv;
    const int vcol = lane & (64 / S - 1), vsub = lane / (64 / S);
    const unsigned vlane = 4 * vsub * vw + vcol, srow = lane & (ROWS - 1);
    auto load_v = [&](int64_t slot) {
      const unsigned* src = p.vc + slot * vw;              // (rows by their scalar address, the lane's part of it a constant)
      if (vcol < vw) {
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
          for (int k = 0; k < 4; ++k) vreg[st][k] = (src + (4 * S * st + k) * vw)[vlane];
      }
      smk = (p.km + slot)[srow];
      smv = (p.vm + slot)[srow];
    };
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int k = 0; k < 4; ++k) vreg[st][k] = 0;

    bool bad0, bad1, bad2, badv = false;                   // of tiles t, t + 1, t + 2, t - 1
    int pg0 = page_of(t0, bad0);
    load_k(slot_of(t0, pg0));
    load_v(slot_of(t0, pg0));
    int pg1 = page_of(t0 + 1, bad1), pg2 = page_of(t0 + 2, bad2);

    // ---- fold the query into B: row m of an A fragment is (head m / 16 of the block's two, column (pair, cos or sin)), a lane has 8
    // values of r
    h16x8 F[MB][NKS];
    float hs;                                              // (softmax lane: head lane >> 4) factor of the finished product
    {
      // the query is scaled to 16 .. 32 by a power of two, so that the fold's rounding to fp16 (2^-11 of each element: a score is a
      // sum of 128 Rk independent ones) meets no subnormals; hs takes the factor back (2^10: the latents are held as (c - z) 2^-10)
      const int e = n & 3, pair = 8 * w + 4 * ((n >> 3) & 1) + 2 * ((n >> 2) & 1) + (e >> 1);
      const h16x8* frag = reinterpret_cast<const h16x8*>(p.bfrag) + ((int64_t)(gv * 8 + w) * MB * NKS) * 64 + lane;
      const h16* q = p.q + (int64_t)b * p.sq_b + (int64_t)h0 * p.sq_h;
      const int hq = min(lane >> 4, nh - 1);
      const h16x8 q8 = *reinterpret_cast<const h16x8*>(q + hq * p.sq_h + 8 * (lane & 15));
      h16 qa[MB], qb[MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const h16* qr = q + min(2 * mb + (n >> 4), nh - 1) * p.sq_h + pair;
        qa[mb] = qr[0];
        qb[mb] = qr[64];
      }
      float big = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) big = fmaxf(big, fabsf((float)q8[d]));
      big = row_max16(big);
      int ex = 0;                                          // exponent of the largest, less 4
      if (big > 0.f && big < INFINITY) ex = (int)(__builtin_bit_cast(unsigned, big) >> 23) - 131;
      hs = p.scale * __builtin_bit_cast(float, (unsigned)(ex + 137) << 23);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const int e0 = __builtin_amdgcn_readlane(ex, 32 * mb), e1 = __builtin_amdgcn_readlane(ex, 32 * mb + 16);
        const float f = __builtin_bit_cast(float, (unsigned)(127 - ((n >> 4) ? e1 : e0)) << 23);
        const float q1 = (float)qa[mb] * f, q2 = (float)qb[mb] * f;
        const float own_f = (e & 1) ? -q1 : q1;
#pragma unroll
        for (int kb = 0; kb < NKS; ++kb) {
          // lanes of a (cos, sin) pair hold B[r, i] and B[r, i + 64]: each takes the other's from its neighbour
          const u32x4 own = __builtin_bit_cast(u32x4, frag[(mb * NKS + kb) * 64]);
          u32x4 oth;
#pragma unroll
          for (int d = 0; d < 4; ++d) oth[d] = __builtin_amdgcn_update_dpp(0, own[d], 0xB1, 0xf, 0xf, false);   // quad_perm [1, 0, 3, 2]
          const h16x8 a = __builtin_bit_cast(h16x8, own), c = __builtin_bit_cast(h16x8, oth);
#pragma unroll
          for (int d = 0; d < 8; ++d) F[mb][kb][d] = (h16)fmaf((float)a[d], own_f, (float)c[d] * q2);
        }
      }
    }

    // ---- rotation state: cos / sin of this lane's 4 pairs at position (block's first) + n, and (in LDS) of a step of 32
    float tc[4], ts[4];
    auto turn = [&](double a, float& c, float& s) {        // v_sin / v_cos take revolutions: off by 1.2e-7 at most
      const double rev = a * 0.15915494309189533577;
      const float f = (float)(rev - rint(rev));
      c = __builtin_amdgcn_cosf(f);
      s = __builtin_amdgcn_sinf(f);
    };
    auto start_angles = [&](int t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double wi = p.inv_freq[8 * w + 4 * (i >> 1) + 2 * hi + (i & 1)];
        turn((double)((int64_t)t * TILE + n - qp) * wi, tc[i], ts[i]);
      }
    };
    if (n < 4) {
      float c, s;
      turn(32.0 * (double)p.inv_freq[8 * w + 4 * (n >> 1) + 2 * hi + (n & 1)], c, s);
      float* o = reinterpret_cast<float*>(smem + L::STEP) + w * 16 + hi * 8 + n;
      o[0] = c;
      o[4] = s;
    }

    // eight codes -> fp16 (c - z) 2^-10, exactly for whole z: the bits of a code in the low bits of a half are the subnormal c 2^-24,
    // four bits up c 2^-20; one packed multiply-add scales it and takes z off.  Order in the word pair: nibbles 0 4 | 1 5 | 2 6 | 3 7.
    // (Subnormals straight into the matrix unit, and z taken off at the end, would be less work: but it aligns their products as if
    // they were normal, and loses bits of the small ones: errors of 2^-19 of a sum, measured.)
    const h16x2 m0 = {(h16)16384.f, (h16)16384.f}, m1 = {(h16)1024.f, (h16)1024.f};
    auto scaled = [&](unsigned bits, h16x2 mul, h16x2 z) { return __builtin_elementwise_fma(__builtin_bit_cast(h16x2, bits), mul, z); };
    auto dequant_k = [&](int buf) {
      const h16x2 meta = __builtin_bit_cast(h16x2, kmeta);
      const h16 mz = meta[1] * (h16)(-0.0009765625f);
      const h16x2 z2 = {mz, mz};
      char* dst = smem + buf * (TILE * L::XS) + (ROWS * w + krow) * L::XS + kpart * UL * 16;
#pragma unroll
      for (int i = 0; i < UL; ++i) {
        const unsigned v = kreg[i], v8 = v >> 8;
        u32x4 o;
        o[0] = __builtin_bit_cast(unsigned, scaled(v & 0x000F000Fu, m0, z2));
        o[1] = __builtin_bit_cast(unsigned, scaled(v & 0x00F000F0u, m1, z2));
        o[2] = __builtin_bit_cast(unsigned, scaled(v8 & 0x000F000Fu, m0, z2));
        o[3] = __builtin_bit_cast(unsigned, scaled(v8 & 0x00F000F0u, m1, z2));
        *reinterpret_cast<u32x4*>(dst + 16 * i) = o;
      }
    };
    dequant_k(t0 & 1);
    load_k(slot_of(t0 + 1, pg1));
    start_angles(t0);

    // ---- running state of this wave's positions (softmax lane: head lane >> 4, position lane & 15)
    float m = -INFINITY, lsum = 0.f, vn = 0.f;
    f32x4 acc[8];                                          // [column of the lane's 8][head], times 2^-10 2^15 / vn
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();

    // scores of tile t, this wave's pairs; then the codes of tile t + 1 and the loads of t + 2
    auto scores = [&](int t) {
      const int buf = t & 1;
      if (t != t0 && ((t - t0) & 31) == 0) start_angles(t);
      // A unit is one 32-position block of one pair of heads: NKS dependent matrix instructions, then its dot products in the shadow
      // of the next unit's
      constexpr int U = NB * MB;
      h16x8 x[NKS];
      f32x16 y[2];
      float part[2][NH];
      const char* const xt = smem + buf * (TILE * L::XS) + n * L::XS + hi * 16;
      auto load_x = [&](int nb) {
#pragma unroll
        for (int kb = 0; kb < NKS; ++kb) x[kb] = *reinterpret_cast<const h16x8*>(xt + 32 * nb * L::XS + kb * 32);
      };
      auto product = [&](int u) {
        f32x16 v = {};
#pragma unroll
        for (int kb = 0; kb < NKS; ++kb) v = __builtin_amdgcn_mfma_f32_32x32x16_f16(F[u % MB][kb], x[kb], v, 0, 0, 0);
        y[u & 1] = v;
        if (u % MB == MB - 1 && u / MB + 1 < NB) load_x(u / MB + 1);
      };
      load_x(0);
      product(0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int nb = u / MB, mb = u % MB;
        if (u + 1 < U) product(u + 1);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s0 = fmaf(y[u & 1][8 * d + 2 * i], tc[i], s0);
            s1 = fmaf(y[u & 1][8 * d + 2 * i + 1], ts[i], s1);
          }
          part[nb & 1][2 * mb + d] = s0 + s1;
        }
        if (mb == MB - 1) {
          const f32x4 rc = step[0], rs = step[1];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float c = tc[i];
            tc[i] = c * rc[i] - ts[i] * rs[i];
            ts[i] = c * rs[i] + ts[i] * rc[i];
          }
          if (nb & 1) {
#pragma unroll
            for (int j = 0; j < NH; ++j) {                 // the two halves of a position's columns; lane = position of the 64
              const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, part[0][j]),
                                                               __builtin_bit_cast(unsigned, part[1][j]), false, false);
              const unsigned lo = sw[0], up = sw[1];       // (plain values first: a bit cast of a vector's element takes element 0)
              red[((buf * 8 + w) * 4 + j) * TILE + 32 * (nb - 1) + lane] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, up);
            }
          }
        }
        if (u + 1 < U) {
#pragma unroll
          for (int kb = 0; kb < NKS; ++kb) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                 // one matrix instruction,
            __builtin_amdgcn_sched_group_barrier(0x002, (32 + NKS - 1) / NKS, 0);   // its share of the vector instructions
          }
        }
      }
      if (t + 1 < t1) dequant_k(buf ^ 1);
      if (t + 2 < t1) load_k(slot_of(t + 2, pg2));
    };

    // softmax and values of tile t (its scores are complete), this wave's positions; then the loads of tile t + 1
    auto values = [&](int t) {
      const int buf = t & 1;
      const int head = lane >> 4, pos = lane & 15;
      const int hsafe = NH == 4 ? head : head & (NH - 1), psafe = pos & (ROWS - 1);
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += red[((buf * 8 + k) * 4 + hsafe) * TILE + ROWS * w + psafe];
      const h16x2 mk = __builtin_bit_cast(h16x2, smk), mv = __builtin_bit_cast(h16x2, smv);
      const bool valid = pos < ROWS && t * TILE + ROWS * w + pos < rows && head < NH;
      s *= (float)mk[0] * hs;
      if (badv) s = NAN;
      if (!valid) s = -INFINITY;
      const float mn = fmaxf(m, row_max16(s));
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      const float pr = __builtin_amdgcn_exp2f(s - ref);
      // Weights: probability times the row's value scale, over the largest scale so far (its power of two) and times 2^15, in fp16:
      // 2^-11 of each weight down to 2^-29 of the largest.
      const float sv = valid ? (float)mv[0] : 0.f;
      const float top = row_max16(fabsf(sv));
      const float vp = fmaxf(vn, __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, top) + 0x7fffffu) & 0x7f800000u));
      const float rv = vp > 0.f ? 32768.f * __builtin_amdgcn_rcpf(vp) : 0.f;      // (of a power of two: exact)
      const h16 wt = (h16)(pr * (sv * rv));
      const float shrink = alpha * vn * rv * (1.f / 32768.f);
      const bool moved = mn != m || vp != vn;
      lsum = lsum * alpha + pr;
      m = mn;
      vn = vp;
      wgt[lane] = wt;
      if (lane < 16) wgt[64 + lane] = valid ? mv[1] * (h16)(-0.0009765625f) : (h16)0.f;
      if (__ballot(moved)) {
#pragma unroll
        for (int j = 0; j < NH; ++j) {
          const float a = lane_value(shrink, 16 * j);
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[c][j] *= a;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const h16x4 a = *reinterpret_cast<const h16x4*>(wgt + (lane & 3) * 16 + 4 * (st * S + vsub));
        const h16x4 z4 = *reinterpret_cast<const h16x4*>(wgt + 64 + 4 * (st * S + vsub));
        const h16x2 z01 = {z4[0], z4[1]}, z23 = {z4[2], z4[3]};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const unsigned sel = half ? 0x07060302u : 0x05040100u;
          const unsigned p01 = __builtin_amdgcn_perm(vreg[st][1], vreg[st][0], sel);
          const unsigned p23 = __builtin_amdgcn_perm(vreg[st][3], vreg[st][2], sel);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const unsigned mask = c & 1 ? 0x00F000F0u : 0x000F000Fu;
            const h16x2 v01 = scaled((c & 2 ? p01 >> 8 : p01) & mask, c & 1 ? m1 : m0, z01);
            const h16x2 v23 = scaled((c & 2 ? p23 >> 8 : p23) & mask, c & 1 ? m1 : m0, z23);
            const h16x4 v = {v01[0], v01[1], v23[0], v23[1]};
            acc[4 * half + c] = __builtin_amdgcn_mfma_f32_4x4x4f16(a, v, acc[4 * half + c], 0, 0, 0);
          }
        }
      }
      if (t + 1 < t1) load_v(slot_of(t + 1, pg0));
    };

    for (int t = t0; t <= t1; ++t) {                       // (the last turn: only the values of the last tile)
      if (w >= 4 && t > t0) values(t - 1);
      if (t < t1) scores(t);
      if (w < 4 && t > t0) values(t - 1);
      badv = bad0;
      pg0 = pg1;
      bad0 = bad1;
      pg1 = pg2;
      bad1 = bad2;
      pg2 = page_of(t + 3, bad2);
      __syncthreads();
    }

    // ---- join the eight waves: slabs of every (wave, subset) through LDS, summed in a fixed order
    float* const slab = reinterpret_cast<float*>(smem);
    float* const stat = reinterpret_cast<float*>(smem + L::STAT);
    lsum = row_sum16(lsum);
    if ((lane & 15) == 0) {
      float* o = stat + (w * 4 + (lane >> 4)) * 4;
      o[0] = m;
      o[1] = vn;
      o[2] = lsum;
    }
    __syncthreads();
    // lane (wave k, head j) of every wave: the maximum of the eight, each wave's factor, the sum of the eight
    {
      const int k = (lane >> 2) & 7, j = lane & 3;
      const float* o = stat + (k * 4 + j) * 4;
      const float mk = o[0];
      float top = mk;
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
      const float a = __builtin_amdgcn_exp2f(mk - (top == -INFINITY ? 0.f : top));
      float sum = a * o[2];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor(sum, x, 64);
      const float mine = a * o[1] * (1.f / 32.f);
      if (w == 0 && lane < 4) {
        stat[128 + j] = sum;
        stat[132 + j] = top;
      }
#pragma unroll
      for (int jj = 0; jj < NH; ++jj) {
        const float f = lane_value(mine, 4 * w + jj);
        if (vcol < vw) {
          float* d = slab + (w * S + vsub) * (PA_SLAB / S) + jj * (512 / S) + 8 * vcol;
          *reinterpret_cast<f32x4*>(d) = f32x4{acc[0][jj] * f, acc[1][jj] * f, acc[2][jj] * f, acc[3][jj] * f};
          *reinterpret_cast<f32x4*>(d + 4) = f32x4{acc[4][jj] * f, acc[5][jj] * f, acc[6][jj] * f, acc[7][jj] * f};
        }
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == nt;                // this workgroup has all of the sequence: the result itself
    const bool poison = pa_bad_len(p, b);
    const int64_t slot = (int64_t)blockIdx.x + b * GV + gv;      // (grows from piece to piece: a slot of its own for each)
    for (int i = tid; i < nh * p.Rv; i += PA_THREADS) {
      const int j = i / p.Rv, c = i - j * p.Rv;
      const float* o = slab + j * (512 / S) + c;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 8 * S; ++k) v += o[k * (PA_SLAB / S)];
      if (whole) p.ctx[((int64_t)b * p.H + h0 + j) * p.Rv + c] = (h16)(poison ? NAN : v / stat[128 + j]);
      else p.part[(int64_t)p.slots * 8 + (slot * 4 + j) * p.Rv + c] = v;
    }
    if (!whole && tid < nh) {
      p.part[(slot * 4 + tid) * 2] = stat[132 + tid];
      p.part[(slot * 4 + tid) * 2 + 1] = stat[128 + tid];
    }
    if (p.direct || at >= end) break;
    if (gv == GV - 1) {
      base = at;
      ++b;
    }
    __syncthreads();                                       // the slabs are read before the next piece's latents overwrite them
  }
  if (p.direct && pa_tiles(p, b) == 0) {                   // an empty sequence: zeros
    const int gv = blockIdx.x % GV, g = gv / p.VG, vg = gv - g * p.VG;
    const int nh = min(NH, p.gs - NH * vg);
    for (int i = tid; i < nh * p.Rv; i += PA_THREADS)
      p.ctx[((int64_t)b * p.H + g * p.gs + NH * vg) * p.Rv + i] = (h16)(pa_bad_len(p, b) ? NAN : 0.f);
  }
}

template <int NKS, int S, int NH>
int pa_launch1(const PagedAttnParams& p, int wgs, hipStream_t stream) {
  auto kern = paged_attn_kernel<NKS, S, NH>;
  const int rc = palu_func_max_lds(reinterpret_cast<const void*>(kern), PaLds<NKS>::BYTES);
  if (rc != PALU_OK) return rc;
  hipLaunchKernelGGL(kern, dim3(wgs), dim3(PA_THREADS), PaLds<NKS>::BYTES, stream, p);
  PALU_LAUNCH_CHECK();
  return PALU_OK;
}
template <int NKS, int S>
int pa_launch2(const PagedAttnParams& p, int heads, int wgs, hipStream_t stream) {
  if constexpr (NKS <= 8)
    if (heads == 4) return pa_launch1<NKS, S, 4>(p, wgs, stream);
  return pa_launch1<NKS, S, 2>(p, wgs, stream);
}
template <int NKS>
int pa_launch3(const PagedAttnParams& p, int subsets, int heads, int wgs, hipStream_t stream) {
  if (subsets == 1) return pa_launch2<NKS, 1>(p, heads, wgs, stream);
  if constexpr (PaLds<NKS>::TILE == 128)                   // (8 positions a wave: two rows of 4 side by side at most)
    if (subsets == 4) return pa_launch2<NKS, 4>(p, heads, wgs, stream);
  return pa_launch2<NKS, 2>(p, heads, wgs, stream);
}
template <int A, int B>
int pa_launch(const PagedAttnParams& p, int nks, int subsets, int heads, int wgs, hipStream_t stream) {
  return nks == A ? pa_launch3<A>(p, subsets, heads, wgs, stream) : pa_launch3<B>(p, subsets, heads, wgs, stream);
}

}  // namespace
