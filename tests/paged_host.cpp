// The paged operators' host checks without a GPU: a context whose code
// objects are not loaded, so that arguments which pass them end in
// IFR_EUNSUPPORTED ("not in the code object").
#include "../inferi_amd/csrc/ctx.h"

extern "C" ifr_ctx *paged_host_ctx() {
    auto *c = new ifr_ctx();
    c->n_cu = 256;
    return c;
}
extern "C" const char *paged_host_error(ifr_ctx *c) { return c->err.c_str(); }
extern "C" void paged_host_free(ifr_ctx *c) { delete c; }
