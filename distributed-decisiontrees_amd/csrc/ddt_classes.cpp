// ddt_classes.cpp -- C-ABI of the class-score operators (include/ddt.h "class scores"): argument checks; the kernels are in ddt_classes.hip.
#include <hip/hip_runtime.h>

#include <cmath>

#include "ddt_classes.h"
#include "ddt_engine_priv.h"

namespace ddt {
namespace {

uint32_t score_bytes(uint32_t dtype) { return dtype == DDT_FP32 ? 4u : 2u; }

// A matrix as the kernels take it: which stride is 1, and the other one.  A single row (class) leaves its stride without meaning: such
// a matrix is either layout, and `want_class_major` says which the caller needs it to be (-1: no preference, row-major if it is both).
struct Layout {
  bool class_major = false;
  uint64_t stride = 0;
};

bool fits(const ddt_scores_t* s, bool class_major) {
  const uint64_t K = s->num_classes, n = s->rows;
  if (class_major) return (s->row_stride == 1 || n <= 1) && (s->class_stride >= n || K == 1);
  return (s->class_stride == 1 || K == 1) && (s->row_stride >= K || n <= 1);
}

int check_scores(ddt_engine* e, const char* what, const ddt_scores_t* s, int want_class_major, Layout* out) {
  if (!s) return fail(e, DDT_EINVAL, "%s: NULL matrix", what);
  if (s->dtype > DDT_BF16) return fail(e, DDT_EINVAL, "%s: dtype %u", what, s->dtype);
  if (s->num_classes == 0 || s->num_classes > DDT_MAX_CLASSES) return fail(e, DDT_EINVAL, "%s: %u classes", what, s->num_classes);
  const uint64_t K = s->num_classes, n = s->rows, limit = uint64_t(1) << 48;
  if (n > limit || s->row_stride > limit || s->class_stride > limit) return fail(e, DDT_EINVAL, "%s: shape out of range", what);
  const bool row_major = fits(s, false), class_major = fits(s, true);
  if (!row_major && !class_major)
    return fail(e, DDT_EINVAL, "%s: strides %llu (rows), %llu (classes) are neither row-major nor class-major without overlap", what,
                (unsigned long long)s->row_stride, (unsigned long long)s->class_stride);
  out->class_major = want_class_major < 0 ? !row_major : want_class_major != 0;
  if (out->class_major ? !class_major : !row_major) return fail(e, DDT_EINVAL, "%s: must be %s", what, out->class_major ? "class-major" : "row-major");
  out->stride = out->class_major ? (K == 1 ? n : s->class_stride) : (n <= 1 ? K : s->row_stride);
  if ((out->class_major ? K : n) > 1 && out->stride > (uint64_t(1) << 60) / (out->class_major ? K : n)) return fail(e, DDT_EINVAL, "%s: shape out of range", what);
  if (n && !s->data) return fail(e, DDT_EINVAL, "%s: NULL data", what);
  if (reinterpret_cast<uintptr_t>(s->data) % score_bytes(s->dtype)) return fail(e, DDT_EINVAL, "%s: data is not aligned to its element", what);
  return DDT_OK;
}

// first byte behind a matrix
uintptr_t end_of(const ddt_scores_t* s, const Layout& l) {
  const uint64_t major = l.class_major ? s->num_classes : s->rows, minor = l.class_major ? s->rows : s->num_classes;
  return reinterpret_cast<uintptr_t>(s->data) + ((major - 1) * l.stride + minor) * score_bytes(s->dtype);
}

// `out` may be `in` itself (an element is read before it is written, by the same thread) but not lie across it
int check_result(ddt_engine* e, const char* what, const ddt_scores_t* in, const Layout& li, const ddt_scores_t* out, Layout* lo) {
  const int rc = check_scores(e, what, out, li.class_major, lo);
  if (rc) return rc;
  if (out->rows != in->rows || out->num_classes != in->num_classes || out->dtype != in->dtype)
    return fail(e, DDT_EINVAL, "%s: shape or type differs from the input's", what);
  if (in->rows == 0) return DDT_OK;
  const uintptr_t a = reinterpret_cast<uintptr_t>(in->data), b = reinterpret_cast<uintptr_t>(out->data);
  if (a < end_of(out, *lo) && b < end_of(in, li) && !(a == b && li.stride == lo->stride))
    return fail(e, DDT_EINVAL, "%s: overlaps the input without being it", what);
  return DDT_OK;
}

int check_temperature(ddt_engine* e, double T) {
  return T >= 1e-3 && T <= 1e3 ? DDT_OK : fail(e, DDT_EINVAL, "temperature %g (0.001 .. 1000)", T);
}

int run(ddt_engine* e, const char* what, hipError_t r) {
  return r == hipSuccess ? DDT_OK : fail(e, DDT_EHIP, "%s -> %s", what, hipGetErrorString(r));
}

int distill(ddt_engine* e, const ddt_scores_t* s, const ddt_teacher_t* t, const float* weight, uint64_t weight_stride, float* d_loss,
            const ddt_scores_t* grad, bool want_grad, void* stream) {
  if (!e) return DDT_EINVAL;
  Layout l, lg;
  int rc = check_scores(e, "student", s, 0, &l);
  if (rc) return rc;
  if (!t) return fail(e, DDT_EINVAL, "NULL teacher");
  if (t->k == 0 || t->k > DDT_MAX_TOP) return fail(e, DDT_EINVAL, "teacher: k %u (1 .. %u)", t->k, (unsigned)DDT_MAX_TOP);
  if (s->rows > 1 && (t->row_stride < t->k || t->row_stride > (uint64_t(1) << 48)))
    return fail(e, DDT_EINVAL, "teacher: row_stride %llu for k %u", (unsigned long long)t->row_stride, t->k);
  if (weight && weight_stride > (uint64_t(1) << 48)) return fail(e, DDT_EINVAL, "row_weight: stride out of range");
  rc = check_temperature(e, t->temperature);
  if (rc) return rc;
  if (want_grad) {
    rc = check_result(e, "gradient", s, l, grad, &lg);
    if (rc) return rc;
  }
  if (s->rows == 0) return DDT_OK;
  if (!t->ids || !t->values) return fail(e, DDT_EINVAL, "teacher: NULL ids or values");
  if (!want_grad && !d_loss) return fail(e, DDT_EINVAL, "NULL loss");
  DeviceGuard dg(e->device);
  if (!dg.ok) return fail(e, DDT_EHIP, "hipSetDevice(%d) failed", e->device);
  DistillArgs a{};
  a.in = s->data, a.n = s->rows, a.stride = l.stride, a.K = s->num_classes, a.k = t->k;
  a.ids = t->ids, a.values = t->values, a.teacher_stride = t->row_stride, a.lse = t->lse;
  a.inv_T = 1.0 / t->temperature, a.scale = (float)(kLog2e / t->temperature);
  a.loss = d_loss;
  if (want_grad) a.weight = weight, a.weight_stride = weight_stride, a.grad = grad->data, a.grad_stride = lg.stride;
  return run(e, "distill", launch_distill(a, s->dtype, reinterpret_cast<hipStream_t>(stream)));
}

}  // namespace
}  // namespace ddt

using namespace ddt;

extern "C" {

int ddt_adjust_scores_device(ddt_engine* e, const ddt_scores_t* in, const ddt_adjust_t* adj, const ddt_scores_t* out, void* stream) {
  if (!e) return DDT_EINVAL;
  Layout li, lo;
  int rc = check_scores(e, "scores", in, -1, &li);
  if (rc) return rc;
  if (!adj) return fail(e, DDT_EINVAL, "NULL adjustment");
  if (out && !fits(out, li.class_major) && fits(out, !li.class_major) && fits(in, !li.class_major)) {  // a single row: take the result's layout
    rc = check_scores(e, "scores", in, !li.class_major, &li);
    if (rc) return rc;
  }
  rc = check_result(e, "adjusted scores", in, li, out, &lo);
  if (rc) return rc;
  const uint64_t limit = uint64_t(1) << 48, words = (in->num_classes + 31u) / 32u;
  if (adj->bias && (adj->bias_row_stride > limit || adj->bias_class_stride > limit)) return fail(e, DDT_EINVAL, "bias: stride out of range");
  if (adj->allowed && adj->allowed_row_stride != 0 && (adj->allowed_row_stride < words || adj->allowed_row_stride > limit))
    return fail(e, DDT_EINVAL, "allowed: row stride %llu for %llu words", (unsigned long long)adj->allowed_row_stride, (unsigned long long)words);
  if (adj->history_len && !adj->history) return fail(e, DDT_EINVAL, "history_len without a history");
  if (adj->history && !adj->history_first) return fail(e, DDT_EINVAL, "history without history_first");
  if (adj->history_len > limit) return fail(e, DDT_EINVAL, "history_len out of range");
  if (in->rows == 0) return DDT_OK;
  DeviceGuard dg(e->device);
  if (!dg.ok) return fail(e, DDT_EHIP, "hipSetDevice(%d) failed", e->device);
  AdjustArgs a{};
  a.in = in->data, a.out = out->data, a.n = in->rows, a.in_stride = li.stride, a.out_stride = lo.stride, a.K = in->num_classes;
  a.bias = adj->bias, a.bias_rs = adj->bias_row_stride, a.bias_cs = adj->bias_class_stride;
  a.allowed = adj->allowed, a.allowed_rs = adj->allowed_row_stride;
  if (adj->history_len) {
    a.history = adj->history, a.first = adj->history_first, a.history_len = adj->history_len, a.prompt = adj->history_prompt;
    a.repetition = adj->repetition, a.frequency = adj->frequency, a.presence = adj->presence;
  }
  return run(e, "adjust", launch_adjust(a, in->dtype, li.class_major, reinterpret_cast<hipStream_t>(stream)));
}

int ddt_top_scores_device(ddt_engine* e, const ddt_scores_t* s, uint32_t k, double temperature, int32_t* d_ids, float* d_values, float* d_lse,
                          void* stream) {
  if (!e) return DDT_EINVAL;
  Layout l;
  int rc = check_scores(e, "scores", s, -1, &l);
  if (rc) return rc;
  if (k == 0 || k > DDT_MAX_TOP) return fail(e, DDT_EINVAL, "k %u (1 .. %u)", k, (unsigned)DDT_MAX_TOP);
  rc = check_temperature(e, temperature);
  if (rc) return rc;
  if (l.class_major && s->num_classes > kTopMaxClassMajor)
    return fail(e, DDT_EUNSUPPORTED, "%u classes in a class-major matrix (at most %u; row-major: %u)", s->num_classes, kTopMaxClassMajor, DDT_MAX_CLASSES);
  if (s->rows == 0) return DDT_OK;
  if (!d_ids || !d_values) return fail(e, DDT_EINVAL, "NULL result buffer");
  DeviceGuard dg(e->device);
  if (!dg.ok) return fail(e, DDT_EHIP, "hipSetDevice(%d) failed", e->device);
  TopArgs a{};
  a.in = s->data, a.n = s->rows, a.stride = l.stride, a.K = s->num_classes, a.k = k;
  a.inv_T = 1.0 / temperature, a.scale = (float)(kLog2e / temperature);
  a.ids = d_ids, a.values = d_values, a.lse = d_lse;
  return run(e, "top", launch_top(a, s->dtype, l.class_major, reinterpret_cast<hipStream_t>(stream)));
}

int ddt_distill_device(ddt_engine* e, const ddt_scores_t* student, const ddt_teacher_t* teacher, float* d_loss, void* stream) {
  return distill(e, student, teacher, nullptr, 0, d_loss, nullptr, false, stream);
}

int ddt_distill_grad_device(ddt_engine* e, const ddt_scores_t* student, const ddt_teacher_t* teacher, const float* row_weight,
                            uint64_t row_weight_stride, float* d_loss, const ddt_scores_t* grad, void* stream) {
  return distill(e, student, teacher, row_weight, row_weight_stride, d_loss, grad, true, stream);
}

}  // extern "C"
