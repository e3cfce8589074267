// mock_classes.cpp -- TEST INFRASTRUCTURE (tests/test_class_scores_host.py): the HIP model and the stand-in engine under the REAL argument
// checks of csrc/ddt_classes.cpp; the launches only note what they were given.
#include "mock_engine.cpp"

#include "ddt_classes.h"

namespace {
int g_launches = 0;
unsigned long long g_note[4] = {};
}  // namespace

namespace ddt {
hipError_t launch_adjust(const AdjustArgs& a, uint32_t, bool class_major, hipStream_t) {
  ++g_launches;
  g_note[0] = class_major, g_note[1] = a.in_stride, g_note[2] = a.out_stride, g_note[3] = a.history != nullptr;
  return hipSuccess;
}
hipError_t launch_top(const TopArgs& a, uint32_t, bool class_major, hipStream_t) {
  ++g_launches;
  g_note[0] = class_major, g_note[1] = a.stride, g_note[2] = a.K, g_note[3] = a.k;
  return hipSuccess;
}
hipError_t launch_distill(const DistillArgs& a, uint32_t, hipStream_t) {
  ++g_launches;
  g_note[0] = a.grad != nullptr, g_note[1] = a.stride, g_note[2] = a.grad_stride, g_note[3] = a.weight_stride;
  return hipSuccess;
}
}  // namespace ddt

extern "C" {
int mock_launches() { return g_launches; }
unsigned long long mock_note(int i) { return g_note[i]; }
const char* mock_error(const ddt_engine* e) { return e->err; }
}
