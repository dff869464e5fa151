// Attention over the 8-bit cache: bf16 queries, head sizes 16 to 64.
#include "cached_attn.h"

int pnfx::attn_bf16_64(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  switch (a.c.D) {
    case 16: return run_rows<bf16, 16>(a, p, st);
    case 32: return run_rows<bf16, 32>(a, p, st);
    case 48: return run_rows<bf16, 48>(a, p, st);
    case 64: return run_rows<bf16, 64>(a, p, st);
  }
  set_error("cached_attn: head size %d", a.c.D);
  return PNFX_EUNSUPPORTED;
}
