/*
 * What gq_paged.h fixes at compile time or computes alike on both sides, for
 * tests/test_paged_parts.py to look at on a CPU.
 */
#include "gq_paged.h"

namespace {
template <int CT, int XT, int HD, int RG>
int lds(int *out) {
  typedef PromptLds<CT, XT, HD, RG, 8 / RG> L;
  const int v[] = {RG, L::QLO, L::SCL, L::USED, L::EXCHANGE, L::ODD, L::BYTES};
  for (int x : v) *out++ = x;
  return sizeof v / sizeof v[0];
}
template <int CT, int XT, int HD>
int lds_of(int *out) {
  int n = lds<CT, XT, HD, 4>(out);
  if constexpr (XT == GQ_BF16) n += lds<CT, XT, HD, 8>(out + n);
  return n;
}
template <int CT>
int lds_of_cache(int *out) {
  int n = lds_of<CT, GQ_F32, 64>(out);
  n += lds_of<CT, GQ_F32, 128>(out + n);
  n += lds_of<CT, GQ_BF16, 64>(out + n);
  return n + lds_of<CT, GQ_BF16, 128>(out + n);
}
} // namespace

/* seven numbers of every prompt kernel's LDS; how many */
extern "C" int parts_prompt_lds(int *out) {
  int n = lds_of_cache<GQ_F32>(out);
  n += lds_of_cache<GQ_BF16>(out + n);
  return n + lds_of_cache<GQ_I8_ROWS>(out + n);
}

extern "C" int parts_len(int before, int n, int max_len) { return pgd_len(before, n, max_len); }
