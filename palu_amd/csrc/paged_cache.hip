// The pages of a 4-bit latent cache that many sequences share: writing rows into them and copying them.
//
// A page holds P consecutive positions of one sequence for all G head groups, as four arrays (include/palu_hip.h):
//   k_codes [N][G][P][Rk / 2] bytes   k_meta [N][G][P][2] fp16   v_codes [N][G][P][Rv / 2]   v_meta [N][G][P][2]
// A group's rows of a page are contiguous, so the attention kernel streams P rows at a time, and a page is one piece of memory
// per array, so that copying it needs no strides.
#include "palu_common.h"

namespace {

static __device__ __forceinline__ float r16(float x) { return (float)(h16)x; }

struct AppendTensor {
  const h16* x;  int64_t sx_t, sx_g;      // rows [T][G][R], element strides
  unsigned* codes;                        // [N][G][P][R / 8] words of eight codes
  unsigned* meta;                         // [N][G][P] (scale, zero) pairs
  int R, lanes;                           // lanes of a row: a power of two >= R / 8, at most 64
};

static __device__ __forceinline__ h16x2 pair_max(h16x2 a, h16x2 b) { return __builtin_elementwise_max(a, b); }

// (maximum, -minimum) of a row over its lanes
static __device__ __forceinline__ h16x2 row_extremes(h16x2 v, int lanes) {
#define STEP(CTRL) v = pair_max(v, __builtin_bit_cast(h16x2, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false)))
  if (lanes > 1) STEP(0xB1);               // quad_perm [1, 0, 3, 2]
  if (lanes > 2) STEP(0x4E);               // quad_perm [2, 3, 0, 1]
  if (lanes > 4) STEP(0x141);              // row_half_mirror: the other four of eight
  if (lanes > 8) STEP(0x140);              // row_mirror: the other eight of sixteen
#undef STEP
  if (lanes > 16) v = pair_max(v, __builtin_bit_cast(h16x2, __shfl_xor(__builtin_bit_cast(int, v), 16, 64)));
  if (lanes > 32) v = pair_max(v, __builtin_bit_cast(h16x2, __shfl_xor(__builtin_bit_cast(int, v), 32, 64)));
  return v;
}

// One row per `lanes` lanes, eight values a lane (v; a lane behind the row's end has none), eight codes a lane.  The arithmetic is
// quantize_tensor's with the reference's defaults (palu/model/modules/quant.py:29-39), bit for bit what palu_quantize_pack writes.
// Three steps are shorter here and give the same bits:
//   w / scale   = q0 + (w - q0 scale) rcp(scale), q0 = w rcp(scale): within 2^-24 of the quotient, which two 11-bit numbers cannot
//                 bring closer than that to a rounding border of fp16 without lying on it, and there the correction is exact;
//   the maxima are taken of the fp16 values, and the steps behind the quotient, each of which rounds to fp16, in fp16.
static __device__ __forceinline__ unsigned quantise8(h16x8 v, bool on, int lanes, h16x2& meta) {
  h16x2 e = {(h16)-INFINITY, (h16)-INFINITY};
  if (on) {
    const h16x2 p[4] = {{v[0], v[1]}, {v[2], v[3]}, {v[4], v[5]}, {v[6], v[7]}};
    const h16x2 hi = pair_max(pair_max(p[0], p[1]), pair_max(p[2], p[3]));
    const h16x2 lo = pair_max(pair_max(-p[0], -p[1]), pair_max(-p[2], -p[3]));
    e = pair_max(h16x2{hi[0], lo[0]}, h16x2{hi[1], lo[1]});
  }
  e = row_extremes(e, lanes);
  const float mx = (float)e[0], mn = -(float)e[1];
  const float range = fmaxf(r16(mx - mn), (float)(h16)1e-5f);
  const float scale = r16(range / 15.0f);
  const float zero = fminf(fmaxf(rintf(r16(-mn / scale)), 0.f), 15.0f);
  const float rs = __builtin_amdgcn_rcpf(scale);
  const h16 z = (h16)zero;
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h16x2 c;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const float w = (float)v[2 * i + d];
      const float q0 = w * rs;
      c[d] = __builtin_elementwise_rint((h16)fmaf(fmaf(-q0, scale, w), rs, q0));
    }
    c = __builtin_elementwise_min(__builtin_elementwise_max(c + h16x2{z, z}, h16x2{(h16)0.f, (h16)0.f}), h16x2{(h16)15.f, (h16)15.f});
    const unsigned u = __builtin_bit_cast(unsigned, c + h16x2{(h16)1024.f, (h16)1024.f}) & 0x000F000Fu;   // 1024 + c: c in the low bits
    bits |= ((u | u >> 12) & 0xFFu) << (8 * i);
  }
  meta = h16x2{(h16)scale, z};
  return bits;
}

// Token rows of one group (blockIdx.y) and one of the two tensors (blockIdx.z): 64 / lanes of them a wave and turn, IT turns, whose rows
// and places are all requested before the first is worked on.
template <int IT>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendTensor a, AppendTensor b, const int* __restrict__ table,
                                                           int64_t st_b, int B, int max_pages, const int* __restrict__ seq,
                                                           const int* __restrict__ pos, int T, int G, int log_p, int n_pages) {
  const AppendTensor& t = blockIdx.z ? b : a;
  const int lane = threadIdx.x & 63, g = blockIdx.y;
  const int sub = lane & (t.lanes - 1), rows = 64 / t.lanes;
  const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (IT * rows) + lane / t.lanes;
  const bool on = 8 * sub < t.R;
  h16x8 v[IT];
  int s[IT], p[IT], page[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int64_t token = first + i * rows;
    v[i] = h16x8{};
    s[i] = p[i] = -1;
    if (token < T) {
      s[i] = seq[token];
      p[i] = pos[token];
      if (on) v[i] = *reinterpret_cast<const h16x8*>(t.x + token * t.sx_t + g * t.sx_g + 8 * sub);
    }
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {                                             // -1: a padding row, or one the table has no page for
    page[i] = -1;
    if (s[i] >= 0 && s[i] < B && p[i] >= 0 && (p[i] >> log_p) < max_pages) page[i] = table[s[i] * st_b + (p[i] >> log_p)];
    if (page[i] >= n_pages) page[i] = -1;
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    h16x2 meta;
    const unsigned bits = quantise8(v[i], on, t.lanes, meta);
    if (page[i] < 0) continue;
    const int64_t slot = (((int64_t)page[i] * G + g) << log_p) + (p[i] & ((1 << log_p) - 1));
    if (on) t.codes[slot * (t.R >> 3) + sub] = bits;
    if (sub == 0) t.meta[slot] = __builtin_bit_cast(unsigned, meta);
  }
}

struct CopyArrays {
  u32x4* p[4];
  int64_t units[4];                       // 16-byte units of a page
};

// One workgroup copies up to 1024 units (16 KB) of one page of one layer: four loads in flight a thread, then four stores.
__global__ __launch_bounds__(256) void paged_copy_kernel(CopyArrays c, const int* __restrict__ src, const int* __restrict__ dst,
                                                         int chunks, int n_pages) {
  const int pair = blockIdx.x / chunks, chunk = blockIdx.x - pair * chunks;
  const int s = src[pair], d = dst[pair];
  if (s < 0 || s >= n_pages || d < 0 || d >= n_pages || s == d) return;
  const int64_t from = (int64_t)blockIdx.y * n_pages + s, to = (int64_t)blockIdx.y * n_pages + d;
  u32x4 v[4];
  u32x4* out[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    int64_t u = (int64_t)chunk * 1024 + k * 256 + threadIdx.x;
    out[k] = nullptr;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (u >= 0 && u < c.units[a]) {
        v[k] = c.p[a][from * c.units[a] + u];
        out[k] = c.p[a] + to * c.units[a] + u;
      }
      u -= c.units[a];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (out[k]) *out[k] = v[k];
}

int log2_exact(int v) {
  for (int i = 0; i < 31; ++i)
    if ((1 << i) == v) return i;
  return -1;
}

int row_lanes(int R) {
  int n = 1;
  while (n * 8 < R) n *= 2;
  return n;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int palu_paged_append_q4(const void* k, int64_t sk_t, int64_t sk_g, const void* v, int64_t sv_t, int64_t sv_g,
                                    void* k_codes, void* k_meta, void* v_codes, void* v_meta, const int* block_table,
                                    int64_t st_b, int B, int max_pages, const int* seq_ids, const int* positions, int T, int G,
                                    int P, int n_pages, int Rk, int Rv, palu_stream_t stream) {
  PALU_REQUIRE(T >= 0 && B >= 0 && max_pages >= 0 && G > 0 && n_pages > 0, PALU_ERR_ARG, "paged_append: bad sizes");
  const int log_p = log2_exact(P);
  PALU_REQUIRE(log_p >= 4, PALU_ERR_UNSUPPORTED, "paged_append: page size must be a power of two >= 16 (got %d)", P);
  PALU_REQUIRE(Rk > 0 && Rk % 8 == 0 && Rk <= 512 && Rv > 0 && Rv % 8 == 0 && Rv <= 512, PALU_ERR_UNSUPPORTED,
               "paged_append: ranks must be multiples of 8 up to 512 (got %d, %d)", Rk, Rv);
  if (T == 0 || B == 0 || max_pages == 0) return PALU_OK;
  PALU_REQUIRE(k && v && k_codes && k_meta && v_codes && v_meta && block_table && seq_ids && positions, PALU_ERR_ARG,
               "paged_append: null pointer");
  PALU_REQUIRE(aligned16(k) && aligned16(v) && sk_t % 8 == 0 && sk_g % 8 == 0 && sv_t % 8 == 0 && sv_g % 8 == 0, PALU_ERR_ARG,
               "paged_append: latent rows must be 16-byte aligned");
  PALU_REQUIRE(aligned16(k_codes) && aligned16(k_meta) && aligned16(v_codes) && aligned16(v_meta), PALU_ERR_ARG,
               "paged_append: the pages must be 16-byte aligned");
  const AppendTensor a = {(const h16*)k, sk_t, sk_g, (unsigned*)k_codes, (unsigned*)k_meta, Rk, row_lanes(Rk)};
  const AppendTensor b = {(const h16*)v, sv_t, sv_g, (unsigned*)v_codes, (unsigned*)v_meta, Rv, row_lanes(Rv)};
  PALU_REQUIRE(G < 65536, PALU_ERR_ARG, "paged_append: too many groups (%d)", G);
  const int most = a.lanes > b.lanes ? a.lanes : b.lanes;
  const int64_t waves = ((int64_t)T * most + 63) / 64;
  // four turns a wave once that still leaves every SIMD of the device its waves
  const bool deep = waves * 2 * G >= (int64_t)palu_num_cus() * 4 * 8 * 4;
  const int64_t wgs = (waves + (deep ? 16 : 4) - 1) / (deep ? 16 : 4);
  dim3 grid((unsigned)wgs, (unsigned)G, 2), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (deep)
    hipLaunchKernelGGL(paged_append_kernel<4>, grid, block, 0, st, a, b, block_table, st_b, B, max_pages, seq_ids, positions, T, G, log_p,
                       n_pages);
  else
    hipLaunchKernelGGL(paged_append_kernel<1>, grid, block, 0, st, a, b, block_table, st_b, B, max_pages, seq_ids, positions, T, G, log_p,
                       n_pages);
  PALU_LAUNCH_CHECK();
  return PALU_OK;
}

extern "C" int palu_paged_copy(void* k_codes, void* k_meta, void* v_codes, void* v_meta, const int* src, const int* dst, int n,
                               int layers, int n_pages, int G, int P, int Rk, int Rv, palu_stream_t stream) {
  PALU_REQUIRE(n >= 0 && layers > 0 && layers < 65536 && n_pages > 0 && G > 0, PALU_ERR_ARG, "paged_copy: bad sizes");
  PALU_REQUIRE(log2_exact(P) >= 4, PALU_ERR_UNSUPPORTED, "paged_copy: page size must be a power of two >= 16 (got %d)", P);
  PALU_REQUIRE(Rk > 0 && Rk % 8 == 0 && Rv > 0 && Rv % 8 == 0, PALU_ERR_UNSUPPORTED,
               "paged_copy: ranks must be multiples of 8 (got %d, %d)", Rk, Rv);
  if (n == 0) return PALU_OK;
  PALU_REQUIRE(k_codes && k_meta && v_codes && v_meta && src && dst, PALU_ERR_ARG, "paged_copy: null pointer");
  PALU_REQUIRE(aligned16(k_codes) && aligned16(k_meta) && aligned16(v_codes) && aligned16(v_meta), PALU_ERR_ARG,
               "paged_copy: the pages must be 16-byte aligned");
  const int64_t gp = (int64_t)G * P;
  CopyArrays c = {{(u32x4*)k_codes, (u32x4*)k_meta, (u32x4*)v_codes, (u32x4*)v_meta},
                  {gp * Rk / 32, gp / 4, gp * Rv / 32, gp / 4}};
  const int64_t chunks = (c.units[0] + c.units[1] + c.units[2] + c.units[3] + 1023) / 1024;
  PALU_REQUIRE(chunks * n < (1ll << 31), PALU_ERR_ARG, "paged_copy: too many pages in one call (%d)", n);
  hipLaunchKernelGGL(paged_copy_kernel, dim3((unsigned)(chunks * n), (unsigned)layers), dim3(256), 0, (hipStream_t)stream, c, src,
                     dst, (int)chunks, n_pages);
  PALU_LAUNCH_CHECK();
  return PALU_OK;
}
