// Attention over the 8-bit cache: bf16 queries, head sizes 80 to 128.
#include "cached_attn.h"

int pnfx::attn_bf16_128(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  switch (a.c.D) {
    case 80: return run_rows<bf16, 80>(a, p, st);
    case 96: return run_rows<bf16, 96>(a, p, st);
    case 112: return run_rows<bf16, 112>(a, p, st);
    case 128: return run_rows<bf16, 128>(a, p, st);
  }
  set_error("cached_attn: head size %d", a.c.D);
  return PNFX_EUNSUPPORTED;
}
