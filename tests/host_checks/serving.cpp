// serving.cpp -- the batched serving calls on a HIP runtime without a device: each line
// read from stdin changes arguments of a call that is right ("name value", or "a+b 1+2" for
// two) and gives the status, and the kernels that are launched.
//   serving DIR append|read|attn|probs|verify
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <map>
#include <string>

#include "fake_hip.hpp"
#include "gemma_hip.h"
#include "runtime/runtime.hpp"

gh_status gh::noalloc_setup(int) { return GH_OK; }

int main(int argc, char** argv) {
  gh_context* made = nullptr;
  if (argc < 3 || gh_context_init(argv[1], &made) != GH_OK) return 2;
  const std::string call = argv[2];
  char name[96], value[96];
  while (scanf("%95s %95s", name, value) == 2) {
    // (no kernel runs: the addresses only have the right alignment)
    std::map<std::string, double> v = {
        {"ctx", 1}, {"cache", 1}, {"batch", 1}, {"k", 4096}, {"v", 4096}, {"k_scale", 4096}, {"v_scale", 4096},
        {"num_pages", 10}, {"page_tokens", 32}, {"num_kv", 2}, {"head_dim", 64}, {"seq_start", 4096}, {"past", 4096},
        {"pages", 4096}, {"num_seqs", 3}, {"max_pages", 40}, {"num_rows", 20}, {"max_rows", 9}, {"q", 4096}, {"kin", 4096},
        {"vin", 4096}, {"qn", 4096}, {"kn", 4096}, {"out", 12288}, {"q_stride", 512}, {"kv_stride", 512}, {"num_q", 4},
        {"rot", 64}, {"k_eq_v", 0}, {"theta", 10000}, {"eps", 1e-6}, {"scale", 1}, {"window", 0}, {"max_kv", 1000},
        {"work", 4096}, {"bytes", 1 << 30}, {"rows", 3}, {"vocab", 1000}, {"stride", 1000}, {"cap", 30}, {"temp", 1},
        {"draft", 4096}, {"tokens", 4096}, {"n_draft", 20480}, {"u", 4096}, {"pick", 4096}, {"accepted", 4096}, {"max_draft", 3}};
    for (char *n = name, *x = value; n;) {
      char *n2 = strchr(n, '+'), *x2 = n2 ? strchr(x, '+') : nullptr;
      if (n2) *n2++ = 0;
      if (x2) *x2++ = 0;
      if (!v.count(n) || (n2 && !x2)) return 2;
      v[n] = atof(x);
      n = n2;
      x = x2;
    }
    const auto at = [&](const char* n) { return reinterpret_cast<void*>((uintptr_t)v[n]); };
    const auto f = [&](const char* n) { return (float*)at(n); };
    const auto w = [&](const char* n) { return (uint32_t*)at(n); };
    const auto u = [&](const char* n) { return (uint32_t)v[n]; };
    gh_context* ctx = v["ctx"] ? made : nullptr;
    gh_kv8_cache cache{at("k"), at("v"), f("k_scale"), f("v_scale"), u("num_pages"), u("page_tokens"), u("num_kv"), u("head_dim")};
    gh_kv8_batch batch{w("seq_start"), w("past"), w("pages"), u("num_seqs"), u("max_pages"), u("num_rows"), u("max_rows")};
    const gh_kv8_cache* c = v["cache"] ? &cache : nullptr;
    const gh_kv8_batch* b = v["batch"] ? &batch : nullptr;
    const size_t bytes = (size_t)v["bytes"];
    size_t need = 0;
    fake::launches.clear();
    gh_status st = GH_OK;
    if (call == "append")
      st = gh_kv8_append(ctx, c, b, f("q"), f("kin"), f("vin"), u("q_stride"), u("kv_stride"), f("qn"), f("kn"), f("out"),
                         u("num_q"), u("rot"), u("k_eq_v"), (float)v["theta"], (float)v["eps"]);
    else if (call == "read")
      st = gh_kv8_read(ctx, c, b, f("kin"), f("vin"));
    else if (call == "attn") {
      need = gh_kv8_attn_workspace(ctx, c, b, u("num_q"), u("window"), u("max_kv"));
      st = gh_kv8_attn(ctx, c, b, f("q"), f("out"), u("num_q"), (float)v["scale"], u("window"), u("max_kv"), at("work"),
                       bytes == 1 ? need - 1 : bytes);
    } else if (call == "probs") {
      need = gh_logit_probs_workspace(ctx, u("rows"), u("vocab"));
      st = gh_logit_probs(ctx, f("q"), f("out"), u("rows"), u("vocab"), u("stride"), (float)v["cap"], (float)v["temp"],
                          at("work"), bytes == 1 ? need - 1 : bytes);
    } else {
      need = gh_spec_verify_workspace(ctx, u("num_seqs"), u("vocab"));
      st = gh_spec_verify(ctx, f("q"), f("draft"), w("tokens"), w("n_draft"), f("u"), f("pick"), w("out"), w("accepted"),
                          u("num_seqs"), u("max_draft"), u("vocab"), at("work"), bytes == 1 ? need - 1 : bytes);
    }
    printf("%d\t%zu\t%s\t", (int)st, need, st == GH_OK ? "" : gh_last_error());
    for (const auto& l : fake::launches)
      printf("%s %u %u %u %u %u;", l.name.c_str(), l.grid[0], l.grid[1], l.grid[2], l.block, l.lds);
    printf("\n");
  }
  gh_context_deinit(made);
  return 0;
}
