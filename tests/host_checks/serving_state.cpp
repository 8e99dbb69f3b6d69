// serving_state.cpp -- what the batched serving calls leave of the host's HIP state and give
// their kernels, on a HIP runtime without a device.  Linked with --wrap for the two
// calls below.
//   serving_state DIR error none|NAME    the error that is pending after a call, of one before it
//   serving_state DIR split PAGES TOKENS  parts, and steps of each, of attention over a table of PAGES pages
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <string>

#include "common/kv8_args.h"
#include "gemma_hip.h"
#include "runtime/runtime.hpp"

gh_status gh::noalloc_setup(int) { return GH_OK; }

namespace {
hipError_t pending = hipSuccess;
int missing = 0;  // lookups that find nothing
Kv8AttnArgs seen{};
}  // namespace

extern "C" {
hipError_t hipPeekAtLastError() { return pending; }
hipError_t hipGetLastError() {
  const hipError_t e = pending;
  pending = hipSuccess;
  return e;
}
hipError_t __real_hipModuleGetFunction(hipFunction_t*, hipModule_t, const char*);
hipError_t __wrap_hipModuleGetFunction(hipFunction_t* f, hipModule_t m, const char* name) {
  if (missing > 0) {
    missing--;
    return pending = hipErrorNotFound;
  }
  return __real_hipModuleGetFunction(f, m, name);
}
hipError_t __real_hipModuleLaunchKernel(hipFunction_t, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned,
                                        hipStream_t, void**, void**);
hipError_t __wrap_hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned by,
                                        unsigned bz, unsigned lds, hipStream_t s, void** args, void** extra) {
  if (strncmp(reinterpret_cast<const char*>(f), "gh_kv8_attn_", 12) == 0) seen = *static_cast<Kv8AttnArgs*>(args[0]);
  return __real_hipModuleLaunchKernel(f, gx, gy, gz, bx, by, bz, lds, s, args, extra);
}
}

int main(int argc, char** argv) {
  gh_context* ctx = nullptr;
  if (argc < 4 || gh_context_init(argv[1], &ctx) != GH_OK) return 2;
  const auto at = [](uintptr_t a) { return reinterpret_cast<void*>(a); };
  // (no kernel runs: the addresses only have the right alignment)
  gh_kv8_cache cache{at(4096), at(4096), (float*)at(4096), (float*)at(4096), 10, 256, 1, 64};
  gh_kv8_batch batch{(uint32_t*)at(4096), (uint32_t*)at(4096), (uint32_t*)at(4096), 1, 40, 1, 1};
  gh_status st;
  if (strcmp(argv[2], "error") == 0) {
    missing = 1;  // (one of the two code objects does not have it)
    pending = strcmp(argv[3], "none") == 0        ? hipSuccess
              : strcmp(argv[3], "not_found") == 0 ? hipErrorNotFound
                                                  : hipErrorInvalidValue;
    st = gh_kv8_read(ctx, &cache, &batch, (float*)at(4096), (float*)at(8192));
    printf("%d %s\n", (int)st, pending == hipSuccess ? "none" : "some");
  } else {
    batch.max_pages = (uint32_t)strtoul(argv[3], nullptr, 10);
    st = gh_kv8_attn(ctx, &cache, &batch, (float*)at(4096), (float*)at(8192), 1, 1.f, 0, (uint32_t)strtoul(argv[4], nullptr, 10),
                     at(4096), (size_t)1 << 40);
    printf("%d %u %u\n", (int)st, seen.nsplit, seen.chunk);
  }
  gh_context_deinit(ctx);
  return 0;
}
