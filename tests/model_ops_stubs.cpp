// What the model operators' entry points (scriptrs_amd/csrc/sfe_ops.cpp) need of a context, without one and
// without a GPU: nothing is launched, calls that pass their checks are counted.
#include <cstdlib>
#include <string>

#include "sfe_ops.hpp"

namespace {
int calls = 0;
std::string message;
}  // namespace

struct sfe_ctx {
  sfe::OpPlans plans;
};

extern "C" sfe_ctx* stub_context() { return new sfe_ctx; }
// Destroys a context; returns how many device buffers it freed.
extern "C" int stub_destroy(sfe_ctx* ctx) {
  int n = 0;
  ctx->plans.close([&](void* p) {
    free(p);
    ++n;
  });
  delete ctx;
  return n;
}
extern "C" int stub_calls() { return calls; }
extern "C" const char* stub_message() { return message.c_str(); }

namespace sfe {

int op_fail(int code, const std::string& msg) {
  message = msg;
  return code;
}
int op_hip_fail(hipError_t, const char* what) { return op_fail(3, what); }
int op_cus(sfe_ctx*) { return 256; }
int op_call(sfe_ctx*, hipStream_t, const char*, hipError_t (*)(void*, int), void*) {
  ++calls;
  return 0;
}
int op_adopt(sfe_ctx* ctx, OpPlan* plan) {
  ctx->plans.adopt(plan, ctx);
  return 0;
}
void op_drop(OpPlan* plan) noexcept {
  if (plan->ctx) plan->ctx->plans.drop(plan);
}
int op_upload(OpPlan* plan, const void*, size_t, size_t room, hipStream_t) {
  if (!plan->ctx->plans.take(room, &plan->buf, &plan->cap)) {
    plan->buf = malloc(room);
    plan->cap = room;
  }
  return 0;
}
int op_scratch(sfe_ctx*, size_t, hipStream_t, void** out) {
  *out = nullptr;
  return 0;
}

hipError_t launch_attn_mask(const uint8_t*, int64_t, uint64_t*, hipStream_t) { return hipSuccess; }
hipError_t launch_attn_zero(const AttnTensor&, int, int, int64_t, int64_t, int64_t, hipStream_t) { return hipSuccess; }
hipError_t launch_attn(const AttnArgs&, int, int, int, hipStream_t) { return hipSuccess; }
hipError_t launch_rotary(const RotaryArgs&, int, bool, int, hipStream_t) { return hipSuccess; }
hipError_t launch_residual(const ResidualArgs&, int, int, hipStream_t) { return hipSuccess; }
size_t beam_scratch_bytes(int, int, int, int) { return 0; }
hipError_t launch_beam_select(const BeamArgs&, int, int, hipStream_t) { return hipSuccess; }
hipError_t launch_beam_reorder(const ReorderArgs&, hipStream_t) { return hipSuccess; }

}  // namespace sfe
