// ddt_classes.h -- kernel arguments of the class-score operators (include/ddt.h "class scores"): ddt_classes.cpp checks the caller's
// arguments and fills these, ddt_classes.hip launches.  Strides are in elements.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ddt {

constexpr double kLog2e = 1.4426950408889634;

struct AdjustArgs {
  const void* in;
  void* out;
  uint64_t n, in_stride, out_stride;  // stride = the one that is not 1: between rows (row-major) or between classes (class-major)
  uint32_t K;
  const float* bias;  // NULL = none
  uint64_t bias_rs, bias_cs;
  const uint32_t* allowed;  // NULL = every class
  uint64_t allowed_rs;
  const int32_t* history;  // NULL = no history
  const int64_t* first;
  uint64_t history_len;
  const int32_t* prompt;
  const float *repetition, *frequency, *presence;
};

struct TopArgs {
  const void* in;
  uint64_t n, stride;
  uint32_t K, k;
  double inv_T;  // 1 / temperature
  float scale;   // log2(e) / temperature
  int32_t* ids;
  float* values;
  float* lse;  // may be NULL
};

struct DistillArgs {
  const void* in;
  uint64_t n, stride;
  uint32_t K, k;
  const int32_t* ids;
  const float* values;
  uint64_t teacher_stride;
  const float* lse;  // NULL: the teacher's mass is on the listed classes
  double inv_T;  // 1 / temperature
  float scale;   // log2(e) / temperature
  const float* weight;  // NULL = 1; only with a gradient
  uint64_t weight_stride;
  float* loss;  // may be NULL with a gradient
  void* grad;   // NULL = loss only
  uint64_t grad_stride;
  bool past_caches;  // set by launch_distill
};

constexpr uint32_t kTopMaxClassMajor = 2048;  // classes of a class-major matrix that the wave-per-row kernel stages in LDS

hipError_t launch_adjust(const AdjustArgs& a, uint32_t dtype, bool class_major, hipStream_t s);
hipError_t launch_top(const TopArgs& a, uint32_t dtype, bool class_major, hipStream_t s);
hipError_t launch_distill(const DistillArgs& a, uint32_t dtype, hipStream_t s);

}  // namespace ddt
