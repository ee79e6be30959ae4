// Paged attention over caches in e4m3 (paged_attention.cuh).
#include "paged_attention.cuh"

namespace b200 {
int pa_run_e4m3(PaArgs& p, int dt, bool pairs, int nc, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st) {
  return pa_run<1>(p, dt, pairs, nc, gen, span, num_sms, ws, need, st);
}
}  // namespace b200
