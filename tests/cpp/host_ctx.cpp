// A context for argument checks without a GPU: rrr_* entry points validate their arguments
// before they touch the device, so a refusal can be tested on a host-made rrr_ctx.
#include "../../recursive-routing-racer-rs_b200/csrc/capi_internal.h"

extern "C" void* host_ctx_new() {
  rrr_ctx* c = new rrr_ctx;
  c->sm_count = 148;
  return c;
}
extern "C" void host_ctx_free(void* c) { delete static_cast<rrr_ctx*>(c); }
