// Decode attention of many sequences over the pages of a 4-bit latent cache: one new token of each of B sequences.
//
//   x_l     = (c_l - z_l) s_l                           the key latent of position l (codes c, fp16 pair (scale s, zero z) a row)
//   score_l = sm_scale <R(pos) q, R(l) (x_l B_h)>       B_h [Rk, 128]: the head's key reconstruction, R(l) the rotation by l
//   ctx     = sum_l softmax(score)_l (v_l - zv_l) sv_l  the head's context in latent space
//
// The rotation of the query is moved to the keys (<R(p) q, R(l) k> = <q, R(l - p) k>), and the query is folded into B:
//   Fc[r, i] = q_i B[r, i] + q_{i+64} B[r, i+64]        Fs[r, i] = q_{i+64} B[r, i] - q_i B[r, i+64]
//   score_l = sum_i cos((l - p) w_i) <x_l, Fc_i> + sin((l - p) w_i) <x_l, Fs_i>
// so no key is ever written down.
#include "palu_common.h"

namespace {

constexpr int PTS = 256;                               // positions of a pass over the sequence = threads

struct PagedAttnParams {
  const h16* q;       int64_t sq_b, sq_h;
  const h16* b;                                        // [H][Rk][128]
  const unsigned* kc; const h16* km;
  const unsigned* vc; const h16* vm;
  const int* table;   int64_t st_b;
  const int* lens;
  const int* qpos;
  const float* inv_freq;
  h16* ctx;
  int B, H, G, max_pages, log_p, n_pages, Rk, Rv;
  float scale;
};

// one workgroup per (sequence, head): the folded query in LDS, a thread scores a position, then a thread sums columns
__global__ __launch_bounds__(PTS) void paged_attn_simple_kernel(PagedAttnParams p) {
  extern __shared__ float smem[];
  float* fold = smem;                                  // [128][Rk]: Fc of pair i in row i, Fs in row 64 + i
  float* prob = fold + 128 * p.Rk;                     // [PTS]
  float* red = prob + PTS;                             // [8]
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y, g = h / (p.H / p.G);
  int len = p.lens[b];
  const bool bad_len = len > (p.max_pages << p.log_p);
  len = min(max(len, 0), p.max_pages << p.log_p);
  const int pos = p.qpos ? p.qpos[b] : 0;
  const h16* q = p.q + b * p.sq_b + h * p.sq_h;
  for (int idx = tid; idx < 64 * p.Rk; idx += PTS) {
    const int r = idx >> 6, i = idx & 63;
    const float b1 = (float)p.b[((int64_t)h * p.Rk + r) * 128 + i], b2 = (float)p.b[((int64_t)h * p.Rk + r) * 128 + 64 + i];
    const float q1 = (float)q[i] * p.scale, q2 = (float)q[i + 64] * p.scale;
    fold[i * p.Rk + r] = q1 * b1 + q2 * b2;
    fold[(64 + i) * p.Rk + r] = q2 * b1 - q1 * b2;
  }
  __syncthreads();
  float m = -INFINITY, sum = 0.f, acc[2] = {0.f, 0.f};
  for (int l0 = 0; l0 < len; l0 += PTS) {
    const int l = l0 + tid;
    float s = -INFINITY;
    if (l < len) {
      const int page = p.table[b * p.st_b + (l >> p.log_p)];
      if (page < 0 || page >= p.n_pages) {
        s = NAN;                                       // a page outside the pool: the sequence's context is NaN, nothing is read
      } else {
        const int64_t slot = (((int64_t)page * p.G + g) << p.log_p) + (l & ((1 << p.log_p) - 1));
        const float sc = (float)p.km[2 * slot], z = (float)p.km[2 * slot + 1];
        s = 0.f;
        for (int i = 0; i < 64; ++i) {
          float yc = 0.f, ys = 0.f;
          for (int u = 0; u < p.Rk / 8; ++u) {
            const unsigned w = p.kc[slot * (p.Rk / 8) + u];
            for (int e = 0; e < 8; ++e) {
              const float x = (float)((w >> (4 * e)) & 15) - z;
              yc = fmaf(x, fold[i * p.Rk + 8 * u + e], yc);
              ys = fmaf(x, fold[(64 + i) * p.Rk + 8 * u + e], ys);
            }
          }
          const double a = (double)(l - pos) * (double)p.inv_freq[i];
          double sn, cs;
          sincos(a, &sn, &cs);
          s += (float)cs * yc + (float)sn * ys;
        }
        s *= sc;
      }
    }
    float mt = wave_max(s);
    if ((tid & 63) == 0) red[tid >> 6] = mt;
    __syncthreads();
    mt = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mnew = fmaxf(m, mt);
    const float base = mnew == -INFINITY ? 0.f : mnew;
    const float pr = l < len ? __expf(s - base) : 0.f;
    prob[tid] = pr;
    const float st = wave_sum(pr);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = st;
    __syncthreads();
    const float alpha = m == -INFINITY ? 0.f : __expf(m - base);
    sum = sum * alpha + red[0] + red[1] + red[2] + red[3];
    for (int k = 0; k < 2; ++k) {
      const int col = tid + k * PTS;
      if (col >= p.Rv) break;
      acc[k] *= alpha;
      for (int j = 0; j < min(PTS, len - l0); ++j) {
        const int page = p.table[b * p.st_b + ((l0 + j) >> p.log_p)];
        if (page < 0 || page >= p.n_pages) {
          acc[k] = NAN;
          continue;
        }
        const int64_t slot = (((int64_t)page * p.G + g) << p.log_p) + ((l0 + j) & ((1 << p.log_p) - 1));
        const unsigned w = p.vc[slot * (p.Rv / 8) + (col >> 3)];
        const float x = ((float)((w >> (4 * (col & 7))) & 15) - (float)p.vm[2 * slot + 1]) * (float)p.vm[2 * slot];
        acc[k] = fmaf(prob[j], x, acc[k]);
      }
    }
    m = mnew;
    __syncthreads();
  }
  for (int k = 0; k < 2; ++k) {
    const int col = tid + k * PTS;
    if (col < p.Rv)
      p.ctx[((int64_t)b * p.H + h) * p.Rv + col] = (h16)(bad_len ? NAN : len == 0 ? 0.f : acc[k] / sum);
  }
}

}  // namespace

extern "C" size_t palu_paged_b_bytes(int H, int G, int R) {
  if (H <= 0 || G <= 0 || H % G || R <= 0 || R % 8 || R > 256) return 0;
  return (size_t)H * R * 128 * 2;
}

extern "C" int palu_paged_prepare_b(const void* b, int H, int G, int R, int D, void* out, palu_stream_t stream) {
  PALU_REQUIRE(D == 128, PALU_ERR_UNSUPPORTED, "paged_prepare_b: head_dim must be 128 (got %d)", D);
  PALU_REQUIRE(palu_paged_b_bytes(H, G, R), PALU_ERR_UNSUPPORTED,
               "paged_prepare_b: need H %% G == 0 and a group rank that is a multiple of 8 up to 256 (got H=%d G=%d R=%d)", H, G, R);
  PALU_REQUIRE(b && out, PALU_ERR_ARG, "paged_prepare_b: null pointer");
  if (hipMemcpyAsync(out, b, palu_paged_b_bytes(H, G, R), hipMemcpyDeviceToDevice, (hipStream_t)stream) != hipSuccess) {
    palu_set_error("paged_prepare_b: copy failed");
    return PALU_ERR_LAUNCH;
  }
  return PALU_OK;
}

extern "C" size_t palu_paged_attn_workspace_bytes(int B, int H, int G, int max_pages, int P, int Rk, int Rv) {
  (void)B, (void)H, (void)G, (void)max_pages, (void)P, (void)Rk, (void)Rv;
  return 16;
}

extern "C" int palu_paged_attn_q4(const void* q, int64_t sq_b, int64_t sq_h, const void* bfrag, const void* k_codes,
                                  const void* k_meta, const void* v_codes, const void* v_meta, const int* block_table, int64_t st_b,
                                  int max_pages, const int* seq_lens, const int* q_positions, const float* inv_freq, void* ctx,
                                  void* workspace, int B, int H, int G, int D, int P, int n_pages, int Rk, int Rv, float sm_scale,
                                  palu_stream_t stream) {
  PALU_REQUIRE(D == 128, PALU_ERR_UNSUPPORTED, "paged_attn: head_dim must be 128 (got %d)", D);
  PALU_REQUIRE(B >= 0 && B < 65536 && H > 0 && G > 0 && H % G == 0 && max_pages >= 0 && n_pages > 0, PALU_ERR_ARG,
               "paged_attn: bad sizes");
  int log_p = -1;
  for (int i = 4; i < 16; ++i)
    if ((1 << i) == P) log_p = i;
  PALU_REQUIRE(log_p > 0, PALU_ERR_UNSUPPORTED, "paged_attn: page size must be a power of two >= 16 (got %d)", P);
  PALU_REQUIRE(Rk > 0 && Rk % 8 == 0 && Rk <= 256 && Rv > 0 && Rv % 8 == 0 && Rv <= 512, PALU_ERR_UNSUPPORTED,
               "paged_attn: group ranks must be multiples of 8, up to 256 (keys) and 512 (values) (got %d, %d)", Rk, Rv);
  PALU_REQUIRE((int64_t)max_pages * P < (1ll << 30), PALU_ERR_ARG, "paged_attn: a sequence may have 2^30 positions at most");
  if (B == 0) return PALU_OK;
  PALU_REQUIRE(q && bfrag && k_codes && k_meta && v_codes && v_meta && (block_table || max_pages == 0) && seq_lens && inv_freq && ctx &&
                   workspace, PALU_ERR_ARG, "paged_attn: null pointer");
  PagedAttnParams p = {(const h16*)q, sq_b, sq_h, (const h16*)bfrag, (const unsigned*)k_codes, (const h16*)k_meta,
                       (const unsigned*)v_codes, (const h16*)v_meta, block_table, st_b, seq_lens, q_positions, inv_freq, (h16*)ctx,
                       B, H, G, max_pages, log_p, n_pages, Rk, Rv, sm_scale};
  const int lds = (128 * Rk + PTS + 8) * 4;
  const int rc = palu_func_max_lds((const void*)paged_attn_simple_kernel, lds);
  if (rc != PALU_OK) return rc;
  hipLaunchKernelGGL(paged_attn_simple_kernel, dim3(H, B), dim3(PTS), lds, (hipStream_t)stream, p);
  PALU_LAUNCH_CHECK();
  return PALU_OK;
}
