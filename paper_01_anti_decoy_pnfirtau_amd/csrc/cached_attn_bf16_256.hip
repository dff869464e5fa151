// Attention over the 8-bit cache: bf16 queries, head sizes 144 to 256.
#include "cached_attn.h"

int pnfx::attn_bf16_256(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  switch (a.c.D) {
    case 144: return run_rows<bf16, 144>(a, p, st);
    case 160: return run_rows<bf16, 160>(a, p, st);
    case 176: return run_rows<bf16, 176>(a, p, st);
    case 192: return run_rows<bf16, 192>(a, p, st);
    case 208: return run_rows<bf16, 208>(a, p, st);
    case 224: return run_rows<bf16, 224>(a, p, st);
    case 240: return run_rows<bf16, 240>(a, p, st);
    case 256: return run_rows<bf16, 256>(a, p, st);
  }
  set_error("cached_attn: head size %d", a.c.D);
  return PNFX_EUNSUPPORTED;
}
