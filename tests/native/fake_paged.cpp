/*
 * A context on the CPU for the host side of the paged entry points: what they
 * ask of the context, the HIP calls they make, and a record of their launches.
 * tests/test_paged_host.py links it with gq_paged.hip in place of the HIP
 * runtime and the rest of the library.
 */
#include <stdio.h>
#include <stdlib.h>

#include <string>

#include "gq_internal.h"

struct gq_ctx {
  std::string err;
};

namespace {
gq_ctx ctx;
long launches;
unsigned long long blocks;
int device;
size_t ws_bytes;
bool refuse_ws;
void *ws;
} // namespace

extern "C" {
gq_ctx *fake_ctx() { return &ctx; }
const char *fake_error() { return ctx.err.c_str(); }
void fake_reset(int refuse) {
  ctx.err.clear(), launches = 0, blocks = 0, device = 0, ws_bytes = 0, refuse_ws = refuse != 0;
}
long fake_launches() { return launches; }
unsigned long long fake_blocks() { return blocks; }
int fake_device() { return device; }
size_t fake_ws() { return ws_bytes; }
void fake_set_device(int d) { device = d; }

hipError_t hipGetDevice(int *d) {
  *d = device;
  return hipSuccess;
}
hipError_t hipSetDevice(int d) {
  device = d;
  return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipLaunchKernel(const void *, dim3 g, dim3, void **, size_t, hipStream_t) {
  launches++, blocks += (unsigned long long)g.x * g.y * g.z;
  return device == 3 ? hipSuccess : hipErrorInvalidDevice; /* the context's device */
}
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t);
hipError_t __hipPopCallConfiguration(dim3 *, dim3 *, size_t *, hipStream_t *);
void **__hipRegisterFatBinary(void *) { return nullptr; }
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, void *, void *, int *) {}
void __hipUnregisterFatBinary(void *) {}
}

static dim3 cfg_g, cfg_b;
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) {
  cfg_g = g, cfg_b = b;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *s, hipStream_t *st) {
  *g = cfg_g, *b = cfg_b, *s = 0, *st = nullptr;
  return hipSuccess;
}

GqCtxInfo gq_ctx_info(const gq_ctx *) { return GqCtxInfo{3, 256, nullptr}; }
int gq_ctx_fail(gq_ctx *c, int code, const char *msg) {
  c->err = msg;
  return code;
}
void *gq_ctx_paged_ws(gq_ctx *, size_t bytes) {
  ws_bytes = bytes;
  if (refuse_ws) return nullptr;
  if (!ws) ws = aligned_alloc(256, 256);
  return ws;
}
