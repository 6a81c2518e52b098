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

// One row per `lanes` lanes, eight values a lane: one 16-byte load, the row's minimum and maximum over its lanes, eight codes, one
// word stored.  The arithmetic is quantize_tensor's with the reference's defaults (palu/model/modules/quant.py:29-39), bit for bit
// what palu_quantize_pack writes; two steps are shorter here and give the same bits:
//   w / scale   = q0 + (w - q0 scale) rcp(scale), q0 = w rcp(scale): within 2^-24 of the quotient, which two 11-bit numbers cannot
//                 bring closer than that to a rounding border of fp16 without lying on it, and there the correction is exact;
//   the fp16 rounding of (code + zero) moves only sums beyond 2048, and those are clamped to the ends of 0 .. 15 either way.
static __device__ __forceinline__ void append_row(const AppendTensor& t, int64_t token, int g, int64_t slot, int sub) {
  const bool on = 8 * sub < t.R;
  h16x8 v = {};
  if (on) v = *reinterpret_cast<const h16x8*>(t.x + token * t.sx_t + g * t.sx_g + 8 * sub);
  float mx = -INFINITY, mn = INFINITY;
  if (on) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mx = fmaxf(mx, (float)v[e]);
      mn = fminf(mn, (float)v[e]);
    }
  }
  for (int o = t.lanes >> 1; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    mn = fminf(mn, __shfl_xor(mn, o, 64));
  }
  const float range = fmaxf(r16(mx - mn), (float)(h16)1e-5f);
  const float scale = r16(range / 15.0f);
  const float zero = fminf(fmaxf(rintf(r16(-mn / scale)), 0.f), 15.0f);
  const float rs = __builtin_amdgcn_rcpf(scale);
  unsigned bits = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float w = (float)v[e];
    const float q0 = w * rs;
    const float q1 = fmaf(fmaf(-q0, scale, w), rs, q0);
    const float c = fminf(fmaxf(rintf(r16(q1)) + zero, 0.f), 15.0f);
    bits |= (unsigned)c << (4 * e);
  }
  if (on) t.codes[slot * (t.R >> 3) + sub] = bits;
  if (sub == 0) {
    const h16x2 m = {(h16)scale, (h16)zero};
    t.meta[slot] = __builtin_bit_cast(unsigned, m);
  }
}

// rows [0, T G) are the key rows, [T G, 2 T G) the value rows; a wave takes 64 / lanes rows of one of the two
__global__ __launch_bounds__(256) void paged_append_kernel(AppendTensor a, AppendTensor b, const int* __restrict__ table,
                                                           int64_t st_b, int B, int max_pages, const int* __restrict__ seq,
                                                           const int* __restrict__ pos, int64_t rows, int64_t waves_a, int G,
                                                           int log_p, int n_pages) {
  const int lane = threadIdx.x & 63;
  int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const bool second = wave >= waves_a;
  if (second) wave -= waves_a;
  const AppendTensor& t = second ? b : a;
  const int sub = lane & (t.lanes - 1);
  const int64_t row = wave * (64 / t.lanes) + lane / t.lanes;
  if (row >= rows) return;
  const int64_t token = row / G;
  const int g = (int)(row - token * G);
  const int s = seq[token], p = pos[token];
  if (s < 0 || s >= B || p < 0 || (p >> log_p) >= max_pages) return;         // a padding row, or one the table has no place for
  const int page = table[s * st_b + (p >> log_p)];
  if (page < 0 || page >= n_pages) return;
  append_row(t, token, g, (((int64_t)page * G + g) << log_p) + (p & ((1 << log_p) - 1)), sub);
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
  const int64_t rows = (int64_t)T * G;
  const int64_t wa = (rows + 64 / a.lanes - 1) / (64 / a.lanes), wb = (rows + 64 / b.lanes - 1) / (64 / b.lanes);
  const int64_t wgs = (wa + wb + 3) / 4;
  PALU_REQUIRE(wgs < (1ll << 31), PALU_ERR_ARG, "paged_append: too many rows (%lld)", (long long)rows);
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, a, b, block_table, st_b, B,
                     max_pages, seq_ids, positions, rows, wa, G, log_p, n_pages);
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
