// Host side of the paged decode attention: the layout of B, the choice of the kernel's form, and the kernel that joins the pieces
// of a sequence.  The attention itself is paged_attn_kernel.h.
#include "paged_attn_kernel.h"

int palu_paged_attn_launch_lo(const void* params, int nks, int chunks, int heads, int wgs, hipStream_t stream);
int palu_paged_attn_launch_mid(const void* params, int nks, int chunks, int heads, int wgs, hipStream_t stream);
int palu_paged_attn_launch_hi(const void* params, int nks, int chunks, int heads, int wgs, hipStream_t stream);

namespace {

// Joins the pieces of one (sequence, head): 64 columns a workgroup, the pieces dealt over four waves.  Sequences that one
// workgroup had whole are done already; empty ones get their zeros here.
static __global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttnParams p, int W) {
  __shared__ float sh[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int GV = p.G * p.VG;
  const int bg = blockIdx.x, b = bg / GV, gv = bg - b * GV, g = gv / p.VG, vg = gv - g * p.VG;
  const int j = blockIdx.y, nh = min(p.heads, p.gs - p.heads * vg);
  const int c = blockIdx.z * 64 + lane;
  if (j >= nh) return;
  h16* out = p.ctx + ((int64_t)b * p.H + g * p.gs + p.heads * vg + j) * p.Rv;
  const int nt = pa_tiles(p, b);
  if (nt == 0) {
    if (w == 0 && c < p.Rv) out[c] = (h16)(pa_bad_len(p, b) ? NAN : 0.f);
    return;
  }
  const PaLine line = pa_line(p, lane, b);
  const int chunk = pa_chunk(p, line.total, W);
  const int begin = line.front + gv * (nt + PA_FIX);       // the tiles lie at begin + PA_FIX .. begin + PA_FIX + nt - 1
  const int first = (begin + PA_FIX) / chunk, last = (begin + PA_FIX + nt - 1) / chunk;
  const int np = last - first + 1;
  if (np == 1) return;
  const float* stat = p.part + ((int64_t)(first + bg) * 4 + j) * 2;
  const float* val = p.part + (int64_t)p.slots * 8 + ((int64_t)(first + bg) * 4 + j) * p.Rv;
  float top = -INFINITY;
  for (int i = lane; i < np; i += 64) top = fmaxf(top, stat[(int64_t)i * 8]);
  top = wave_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int i = lane; i < np; i += 64) sum += __builtin_amdgcn_exp2f(stat[(int64_t)i * 8] - ref) * stat[(int64_t)i * 8 + 1];
  sum = wave_sum(sum);
  float v = 0.f;
  if (c < p.Rv)
    for (int i = w; i < np; i += 4) v = fmaf(__builtin_amdgcn_exp2f(stat[(int64_t)i * 8] - ref), val[(int64_t)i * 4 * p.Rv + c], v);
  sh[w][lane] = v;
  __syncthreads();
  if (w == 0 && c < p.Rv) out[c] = (h16)(pa_bad_len(p, b) ? NAN : (sh[0][lane] + sh[1][lane] + sh[2][lane] + sh[3][lane]) / sum);
}


// One 16-byte piece a thread: eight values of r of one column of B, in the order in which the kernel finds a word's codes.
__global__ __launch_bounds__(256) void paged_prepare_b_kernel(const h16* __restrict__ b, int G, int gs, int VG, int heads, int R, int nks,
                                                              u32x4* __restrict__ out, int64_t pieces) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= pieces) return;
  const int lane = (int)(idx & 63), kb = (int)((idx >> 6) % nks);
  const int64_t rest = (idx >> 6) / nks;
  const int mbs = heads / 2, mb = (int)(rest % mbs), w = (int)((rest / mbs) & 7), gv = (int)(rest / mbs >> 3);
  const int n = lane & 31, e = n & 3;
  const int g = gv / VG, hl = heads * (gv - g * VG) + 2 * mb + (n >> 4);
  const int col = 8 * w + 4 * ((n >> 3) & 1) + 2 * ((n >> 2) & 1) + (e >> 1) + 64 * (e & 1);
  h16x8 v;
  // 16-byte piece u of a position's row in LDS is word i of part `part` of the row; the last parts are moved back to end with the row,
  // and what they then hold a second time counts for nothing
  const int u = 2 * kb + (lane >> 5), ul = nks / 2, part = u / ul, i = u % ul;
  const int word = min(part * ul, R / 8 - ul) + i;
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    const int r = 8 * word + (d >> 1) + 4 * (d & 1);
    v[d] = hl < gs && word >= part * ul ? b[((int64_t)(g * gs + hl) * R + r) * 128 + col] : (h16)0.f;
  }
  out[idx] = __builtin_bit_cast(u32x4, v);
}

// 16-column blocks of the padded key rank: the forms the kernel exists in
int pa_nks(int R) {
  for (int n : {2, 4, 6, 8, 12, 16})
    if (R <= 16 * n) return n;
  return 0;
}
bool pa_heads_ok(int H, int G, int R) { return H > 0 && G > 0 && H % G == 0 && R > 0 && R % 8 == 0 && R <= 256; }
// heads of a set (see paged_attn_kernel.h), and the sets of a latent group
int pa_heads(int H, int G, int R) { return H / G <= 2 || R > 128 ? 2 : 4; }
int pa_vg(int H, int G, int R) { return (H / G + pa_heads(H, G, R) - 1) / pa_heads(H, G, R); }

struct PaPlan {
  int wgs, slots, min_chunk, direct;
};
// Workgroups of a launch: what the device holds at once, at most one per min_chunk tiles of the longest possible batch.
PaPlan pa_plan(int B, int H, int G, int max_pages, int P, int Rk) {
  PaPlan s;
  const int64_t gv = (int64_t)G * pa_vg(H, G, Rk);
  const int64_t tiles = ((int64_t)max_pages * P + PA_TILE - 1) / PA_TILE;     // of the longest sequence the table has room for
  s.min_chunk = 1;
  s.direct = tiles <= s.min_chunk;
  if (s.direct) {
    s.wgs = (int)(B * gv);
    s.slots = 1;
    return s;
  }
  const int64_t all = B * gv * ((tiles + s.min_chunk - 1) / s.min_chunk);
  const int64_t fit = (int64_t)palu_num_cus();
  s.wgs = (int)(all < fit ? all : fit);
  s.slots = (int)(s.wgs + B * gv);
  return s;
}

}  // namespace

extern "C" size_t palu_paged_b_bytes(int H, int G, int R) {
  return pa_heads_ok(H, G, R) ? (size_t)G * pa_vg(H, G, R) * 8 * (pa_heads(H, G, R) / 2) * pa_nks(R) * 1024 : 0;
}

extern "C" int palu_paged_prepare_b(const void* b, int H, int G, int R, int D, void* out, palu_stream_t stream) {
  PALU_REQUIRE(D == 128, PALU_ERR_UNSUPPORTED, "paged_prepare_b: head_dim must be 128 (got %d)", D);
  PALU_REQUIRE(pa_heads_ok(H, G, R), PALU_ERR_UNSUPPORTED,
               "paged_prepare_b: need H %% G == 0 and a group rank that is a multiple of 8 up to 256 (got H=%d G=%d R=%d)", H, G, R);
  PALU_REQUIRE(b && out && ((uintptr_t)out & 15) == 0, PALU_ERR_ARG, "paged_prepare_b: null or unaligned pointer");
  const int64_t pieces = (int64_t)palu_paged_b_bytes(H, G, R) / 16;
  hipLaunchKernelGGL(paged_prepare_b_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream, (const h16*)b, G,
                     H / G, pa_vg(H, G, R), pa_heads(H, G, R), R, pa_nks(R), (u32x4*)out, pieces);
  PALU_LAUNCH_CHECK();
  return PALU_OK;
}

extern "C" size_t palu_paged_attn_workspace_bytes(int B, int H, int G, int max_pages, int P, int Rk, int Rv) {
  if (B <= 0 || !pa_heads_ok(H, G, Rk) || max_pages <= 0 || P <= 0 || Rv <= 0) return 16;
  const PaPlan s = pa_plan(B, H, G, max_pages, P, Rk);
  return s.direct ? 16 : (size_t)s.slots * (8 + 4 * (size_t)Rv) * 4;
}

extern "C" int palu_paged_attn_q4(const void* q, int64_t sq_b, int64_t sq_h, const void* bfrag, const void* k_codes,
                                  const void* k_meta, const void* v_codes, const void* v_meta, const int* block_table, int64_t st_b,
                                  int max_pages, const int* seq_lens, const int* q_positions, const float* inv_freq, void* ctx,
                                  void* workspace, int B, int H, int G, int D, int P, int n_pages, int Rk, int Rv, float sm_scale,
                                  palu_stream_t stream) {
  PALU_REQUIRE(D == 128, PALU_ERR_UNSUPPORTED, "paged_attn: head_dim must be 128 (got %d)", D);
  PALU_REQUIRE(B >= 0 && B < 65536 && H > 0 && H < 65536 && G > 0 && H % G == 0 && max_pages >= 0 && n_pages > 0, PALU_ERR_ARG,
               "paged_attn: bad sizes");
  int log_p = -1;
  for (int i = 4; i < 16; ++i)
    if ((1 << i) == P) log_p = i;
  PALU_REQUIRE(log_p > 0, PALU_ERR_UNSUPPORTED, "paged_attn: page size must be a power of two from 16 to 32768 (got %d)", P);
  PALU_REQUIRE(Rk > 0 && Rk % 8 == 0 && Rk <= 256 && Rv > 0 && Rv % 8 == 0 && Rv <= 512, PALU_ERR_UNSUPPORTED,
               "paged_attn: group ranks must be multiples of 8, up to 256 (keys) and 512 (values) (got %d, %d)", Rk, Rv);
  PALU_REQUIRE((int64_t)max_pages * P < (1ll << 30), PALU_ERR_ARG, "paged_attn: a sequence may have 2^30 positions at most");
  PALU_REQUIRE((int64_t)B * H * ((int64_t)max_pages * P / 64 + PA_FIX + 1) < (1ll << 31), PALU_ERR_ARG,
               "paged_attn: B * H * max_pages * P must stay below 2^37");
  if (B == 0) return PALU_OK;
  PALU_REQUIRE(q && bfrag && k_codes && k_meta && v_codes && v_meta && (block_table || max_pages == 0) && seq_lens && inv_freq && ctx &&
                   workspace, PALU_ERR_ARG, "paged_attn: null pointer");
  PALU_REQUIRE(((uintptr_t)q & 15) == 0 && sq_b % 8 == 0 && sq_h % 8 == 0 && ((uintptr_t)bfrag & 15) == 0, PALU_ERR_ARG,
               "paged_attn: queries and fragments must be 16-byte aligned");
  const int VG = pa_vg(H, G, Rk), nks = pa_nks(Rk);
  const PaPlan s = pa_plan(B, H, G, max_pages, P, Rk);
  const int heads = pa_heads(H, G, Rk);
  const PagedAttnParams p = {(const h16*)q, sq_b, sq_h, (const h16*)bfrag, (const unsigned*)k_codes, (const unsigned*)k_meta,
                             (const unsigned*)v_codes, (const unsigned*)v_meta, block_table, st_b, seq_lens, q_positions, inv_freq,
                             (h16*)ctx, (float*)workspace, s.slots, B, H, G, H / G, VG, max_pages, log_p, n_pages, Rk, Rv, heads,
                             s.min_chunk, s.direct, sm_scale * 1.44269504088896f};
  const int chunks = (Rv + 127) / 128;
  hipStream_t st = (hipStream_t)stream;
  const int rc = nks <= 4 ? palu_paged_attn_launch_lo(&p, nks, chunks, heads, s.wgs, st)
                 : nks <= 8 ? palu_paged_attn_launch_mid(&p, nks, chunks, heads, s.wgs, st)
                            : palu_paged_attn_launch_hi(&p, nks, chunks, heads, s.wgs, st);
  if (rc != PALU_OK || s.direct) return rc;
  hipLaunchKernelGGL(paged_attn_join_kernel, dim3((unsigned)(B * G * VG), (unsigned)heads, (unsigned)((Rv + 63) / 64)), dim3(256), 0, st, p,
                     s.wgs);
  PALU_LAUNCH_CHECK();
  return PALU_OK;
}
