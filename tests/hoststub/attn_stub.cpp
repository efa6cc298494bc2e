// The attention launchers for the host-only build (see hip_stub.cpp; TEST INFRASTRUCTURE): they keep what the host code hands
// to the kernels, so that a test can look at it.
#include <hip/hip_runtime_api.h>

#include "../../ijah_amd/csrc/attn.h"

namespace {
int launches = 0, attrs = 0;
ijah::KvArgs kv;
ijah::DecArgs dec;
ijah::PromptArgs prompt;
}  // namespace

extern "C" {
hipError_t hipDeviceSynchronize() { return hipSuccess; }
int attnstub_launches() { return launches; }
int attnstub_attrs() { return attrs; }
float attnstub_scale(int which) { return which ? prompt.scale : dec.scale; }
long attnstub_ld(int which) { return which == 0 ? kv.k.ld : which == 1 ? kv.v.ld : which == 2 ? dec.q.ld : prompt.k.ld; }
const void *attnstub_base() { return kv.base; }
}

namespace ijah {
void launch_kv_write(const KvArgs &a, hipStream_t) {
  kv = a;
  launches++;
}
void launch_kv_read(const KvArgs &a, hipStream_t) {
  kv = a;
  launches++;
}
int compute_units() { return 256; }
int decode_grid(int) { return 256; }
void launch_attn_decode(const DecArgs &a, hipStream_t) {
  dec = a;
  launches++;
}
void launch_attn_prompt(const PromptArgs &a, hipStream_t) {
  prompt = a;
  launches++;
}
void init_attn_attrs() { attrs++; }
}  // namespace ijah
