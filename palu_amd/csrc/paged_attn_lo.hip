// paged_attn_kernel (paged_attn_kernel.h) for key ranks up to 2 and 4 blocks of 16 columns; a translation unit of its own so that the
// instances compile side by side.
#include "paged_attn_kernel.h"

int palu_paged_attn_launch_lo(const void* params, int nks, int chunks, int heads, int wgs, hipStream_t stream) {
  return pa_launch<2, 4>(*reinterpret_cast<const PagedAttnParams*>(params), nks, chunks, heads, wgs, stream);
}
