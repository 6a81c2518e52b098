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
  int R, log_lanes, chunks;               // lanes of a row: a power of two up to 16; words of eight values a lane
};

static __device__ __forceinline__ h16x2 pair_max(h16x2 a, h16x2 b) { return __builtin_elementwise_max(a, b); }
static __device__ __forceinline__ h16x2 pair_min(h16x2 a, h16x2 b) { return __builtin_elementwise_min(a, b); }
static __device__ __forceinline__ h16x2 both(h16 a) { return h16x2{a, a}; }

// (maximum, -minimum) of a row over its lanes
static __device__ __forceinline__ h16x2 row_extremes(h16x2 v, int log_lanes) {
#define STEP(CTRL) v = pair_max(v, __builtin_bit_cast(h16x2, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false)))
  if (log_lanes > 0) STEP(0xB1);           // quad_perm [1, 0, 3, 2]
  if (log_lanes > 1) STEP(0x4E);           // quad_perm [2, 3, 0, 1]
  if (log_lanes > 2) STEP(0x141);          // row_half_mirror: the other four of eight
  if (log_lanes > 3) STEP(0x140);          // row_mirror: the other eight of sixteen
#undef STEP
  return v;
}

// The quotient w / s of two fp16 values, rs = rcp(s): within 2^-24 of it, which two 11-bit numbers cannot bring closer than that to a
// rounding border of fp16 without lying on it, and there the correction is exact.  So it rounds to the quotient's fp16.
static __device__ __forceinline__ float quotient(float w, float s, float rs) {
  const float q = w * rs;
  return fmaf(fmaf(-q, s, w), rs, q);
}

// A row's part of one lane, C words of eight values (a word behind the row's end counts for nothing: on[]), to as many words of eight
// codes and the row's pair.  The arithmetic is quantize_tensor's with the reference's defaults (palu/model/modules/quant.py:29-39), bit
// for bit what palu_quantize_pack writes, in fewer steps: the maxima are taken of the fp16 values; the integer next to a quotient x is
// taken by adding 1536 in fp16, whose step is 1 there (from |x| = 512 on it is not the nearest one, but on the right side of the
// clamp, which the zero's 0 .. 15 cannot reach across); clamping comes before the zero, with the borders moved instead; and the
// codes of four values meet as 1024 + a + 16 b, exact in fp16, whose low byte is the byte.
template <int C>
static __device__ __forceinline__ h16x2 quantise(const h16x8 (&v)[C], const bool (&on)[C], int log_lanes, unsigned (&bits)[C]) {
  h16x2 e = both((h16)-INFINITY);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const h16x2 p[4] = {{v[c][0], v[c][1]}, {v[c][2], v[c][3]}, {v[c][4], v[c][5]}, {v[c][6], v[c][7]}};
    const h16x2 hi = pair_max(pair_max(p[0], p[1]), pair_max(p[2], p[3]));
    const h16x2 lo = pair_max(pair_max(-p[0], -p[1]), pair_max(-p[2], -p[3]));
    if (on[c]) e = pair_max(e, pair_max(h16x2{hi[0], lo[0]}, h16x2{hi[1], lo[1]}));
  }
  e = row_extremes(e, log_lanes);
  const float mx = (float)e[0], mn = -(float)e[1];
  const float range = fmaxf(r16(mx - mn), (float)(h16)1e-5f);
  const float scale = r16(range / 15.0f);                                    // (the range may be infinite: a division)
  const float rs = __builtin_amdgcn_rcpf(scale);
  const float zero = fminf(fmaxf(rintf(r16(quotient(-mn, scale, rs))), 0.f), 15.0f);
  const h16x2 low = both((h16)(1536.f - zero)), high = both((h16)(1551.f - zero));
  const h16x2 to_code = both((h16)(zero - 1536.f)), to_byte = both((h16)(zero - 512.f));
#pragma unroll
  for (int c = 0; c < C; ++c) {
    h16x2 y[4];                                                              // values j and j + 4
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const h16x2 q = {(h16)quotient((float)v[c][j], scale, rs), (h16)quotient((float)v[c][j + 4], scale, rs)};
      y[j] = pair_min(pair_max(q + both((h16)1536.f), low), high);
    }
    const h16x2 a = (y[1] + to_code) * both((h16)16.f) + (y[0] + to_byte), b = (y[3] + to_code) * both((h16)16.f) + (y[2] + to_byte);
    bits[c] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x06020400u);
  }
  return h16x2{(h16)scale, (h16)zero};
}

struct AppendPlace {
  const int* table;  int64_t st_b;  int B, max_pages;
  const int *seq, *pos;  int T, G, log_p, n_pages;
};

// IT turns of 64 / lanes token rows of group g each; all rows and places are requested before the first is worked on.
template <int C, int IT>
static __device__ __forceinline__ void append_rows(const AppendTensor& t, const AppendPlace& a, int64_t wave, int g) {
  const int lane = threadIdx.x & 63, sub = lane & ((1 << t.log_lanes) - 1), rows = 64 >> t.log_lanes;
  const int64_t first = wave * (IT * rows) + (lane >> t.log_lanes);
  const int words = t.R >> 3;
  bool on[C];
#pragma unroll
  for (int c = 0; c < C; ++c) on[c] = sub + (c << t.log_lanes) < words;
  h16x8 v[IT][C];
  int s[IT], p[IT], page[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int64_t token = first + i * rows;
    s[i] = p[i] = -1;
#pragma unroll
    for (int c = 0; c < C; ++c) v[i][c] = h16x8{};
    if (token < a.T) {
      s[i] = a.seq[token];
      p[i] = a.pos[token];
      const h16* x = t.x + token * t.sx_t + g * t.sx_g + 8 * sub;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (on[c]) v[i][c] = *reinterpret_cast<const h16x8*>(x + (8 * c << t.log_lanes));
    }
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {                                             // -1: a padding row, or one the table has no page for
    page[i] = -1;
    if (s[i] >= 0 && s[i] < a.B && p[i] >= 0 && (p[i] >> a.log_p) < a.max_pages) page[i] = a.table[s[i] * a.st_b + (p[i] >> a.log_p)];
    if (page[i] >= a.n_pages) page[i] = -1;
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    unsigned bits[C];
    const h16x2 meta = quantise<C>(v[i], on, t.log_lanes, bits);
    if (page[i] < 0) continue;
    const int64_t slot = (((int64_t)page[i] * a.G + g) << a.log_p) + (p[i] & ((1 << a.log_p) - 1));
    unsigned* to = t.codes + slot * words + sub;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (on[c]) to[c << t.log_lanes] = bits[c];
    if (sub == 0) t.meta[slot] = __builtin_bit_cast(unsigned, meta);
  }
}

// One group (blockIdx.y) of one of the two tensors (blockIdx.z).  Sixteen lanes a row at the most: a row of 384 values then fills three
// words of every lane, and the arithmetic of the pair is done for four rows at once.  (A lane per word, 64 lanes a row, left a quarter of
// the wave idle at 384 and worked out every row's pair by itself: 73 us for 16396 tokens of 8 groups x (128 + 384) values, which this
// reads and writes in 38 us: 168 MB at 4.4 TB/s, a large copy's rate being 5.1.  A decode step's 32 rows: 3.4 us, launch and two loads.)
template <int IT>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendTensor k, AppendTensor v, AppendPlace a) {
  const AppendTensor& t = blockIdx.z ? v : k;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  switch (t.chunks) {
    case 1: append_rows<1, IT>(t, a, wave, blockIdx.y); break;
    case 2: append_rows<2, IT>(t, a, wave, blockIdx.y); break;
    case 3: append_rows<3, IT>(t, a, wave, blockIdx.y); break;
    default: append_rows<4, IT>(t, a, wave, blockIdx.y); break;
  }
}

struct CopyArrays {
  u32x4* p[4];
  int64_t units[4];                       // 16-byte units of a page
};

// One workgroup copies up to 1024 units (16 KB) of one page of one layer: four loads in flight a thread, then four stores.  Bound by the
// memory: 1000 pages of 8 x 64 rows (270 MB moved) in 44 us, 6.1 TB/s (part of it from the last-level cache); 9 pages of 32 layers 13 us.
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

int row_log_lanes(int R) {
  int n = 0;
  while (n < 4 && (8 << n) < R) ++n;
  return n;
}

AppendTensor append_tensor(const void* x, int64_t sx_t, int64_t sx_g, void* codes, void* meta, int R) {
  const int n = row_log_lanes(R);
  return {(const h16*)x, sx_t, sx_g, (unsigned*)codes, (unsigned*)meta, R, n, ((R >> 3) + (1 << n) - 1) >> n};
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
  PALU_REQUIRE(G < 65536, PALU_ERR_ARG, "paged_append: too many groups (%d)", G);
  const AppendTensor kt = append_tensor(k, sk_t, sk_g, k_codes, k_meta, Rk), vt = append_tensor(v, sv_t, sv_g, v_codes, v_meta, Rv);
  const AppendPlace at = {block_table, st_b, B, max_pages, seq_ids, positions, T, G, log_p, n_pages};
  const int log_lanes = kt.log_lanes > vt.log_lanes ? kt.log_lanes : vt.log_lanes;
  const int64_t waves = ((int64_t)T + (64 >> log_lanes) - 1) / (64 >> log_lanes);
  // two turns a wave once that still leaves every SIMD of the device its waves
  const bool deep = waves * 2 * G >= (int64_t)palu_num_cus() * 4 * 8 * 2;
  const int64_t wgs = (waves + (deep ? 8 : 4) - 1) / (deep ? 8 : 4);
  dim3 grid((unsigned)wgs, (unsigned)G, 2), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (deep)
    hipLaunchKernelGGL(paged_append_kernel<2>, grid, block, 0, st, kt, vt, at);
  else
    hipLaunchKernelGGL(paged_append_kernel<1>, grid, block, 0, st, kt, vt, at);
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
