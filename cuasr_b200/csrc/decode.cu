// extern "C" boundary of the decoding operators: argument checks, the device the call runs on, launches.
#include <algorithm>

#include "decode_launch.h"

namespace cuasr_b200 {
namespace {

bool is_real(int dtype) { return dtype == CUASR_F32 || dtype == CUASR_F16 || dtype == CUASR_BF16; }
size_t element_bytes(int dtype) { return dtype == CUASR_F32 ? 4 : 2; }
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Makes the device of a call current and sets the caller's back at the end.
class DeviceScope {
 public:
  explicit DeviceScope(int32_t device) {
    if (device == 0) return;
    int now = 0, count = 0;
    ok_ = cudaGetDeviceCount(&count) == cudaSuccess && device <= count && cudaGetDevice(&now) == cudaSuccess;
    if (ok_ && now != device - 1) {
      ok_ = cudaSetDevice(device - 1) == cudaSuccess;
      if (ok_) back_ = now;
    }
  }
  ~DeviceScope() {
    if (back_ >= 0) (void)cudaSetDevice(back_);
  }
  bool ok() const { return ok_; }

 private:
  bool ok_ = true;
  int back_ = -1;
};

int validate_q4(const cuasr_b200_q4_args_t* a) {
  if (a == nullptr) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (!is_real(a->dtype_x) || !is_real(a->dtype_y) || !is_real(a->dtype_scale)) return CUASR_STATUS_ERROR_INVALID_DATA_TYPE;
  if (a->m <= 0 || a->n <= 0 || a->k <= 0 || a->device < 0) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (a->group <= 0 || a->group % 32 != 0) return CUASR_STATUS_ERROR_NOT_SUPPORTED;
  const int64_t groups = (static_cast<int64_t>(a->k) + a->group - 1) / a->group;
  if (a->X == nullptr || a->W == nullptr || a->scales == nullptr || a->Y == nullptr) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (a->ldx < a->k || a->ldw < (static_cast<int64_t>(a->k) + 1) / 2 || a->ld_scales < groups || a->ldy < a->n ||
      (a->zeros != nullptr && a->ld_zeros < groups))
    return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (!aligned(a->X, element_bytes(a->dtype_x)) || !aligned(a->Y, element_bytes(a->dtype_y)) ||
      !aligned(a->scales, element_bytes(a->dtype_scale)))
    return CUASR_STATUS_ERROR_MISALIGNED_OPERAND;
  return q4_fits(*a) ? CUASR_STATUS_SUCCESS : CUASR_STATUS_ERROR_NOT_SUPPORTED;
}

int validate_beam_sizes(const cuasr_b200_beam_args_t* a) {
  if (a == nullptr) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (!is_real(a->dtype)) return CUASR_STATUS_ERROR_INVALID_DATA_TYPE;
  if (a->batch <= 0 || a->beams <= 0 || a->vocab <= 0 || a->keep <= 0 || a->device < 0) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (a->beams > 1024 || a->keep > CUASR_B200_BEAM_MAX_KEEP) return CUASR_STATUS_ERROR_NOT_SUPPORTED;
  if (static_cast<int64_t>(a->batch) * a->beams > (1 << 24)) return CUASR_STATUS_ERROR_NOT_SUPPORTED;
  return CUASR_STATUS_SUCCESS;
}

int validate_beam(const cuasr_b200_beam_args_t* a) {
  const int st = validate_beam_sizes(a);
  if (st != CUASR_STATUS_SUCCESS) return st;
  if (a->logits == nullptr || a->scores == nullptr || a->out_scores == nullptr || a->parents == nullptr || a->tokens == nullptr)
    return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (a->batch_stride < 0 || a->beam_stride < 0 || a->ld_scores < a->beams || a->ld_out_scores < a->keep ||
      a->ld_parents < a->keep || a->ld_tokens < a->keep || (a->finished != nullptr && a->ld_finished < a->beams))
    return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (!aligned(a->logits, element_bytes(a->dtype)) || !aligned(a->scores, 4) || !aligned(a->out_scores, 4) ||
      !aligned(a->parents, 4) || !aligned(a->tokens, 4))
    return CUASR_STATUS_ERROR_MISALIGNED_OPERAND;
  // every search reads its scores before it writes; a search that read another's line would race
  if (a->out_scores == a->scores && a->ld_out_scores != a->ld_scores) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  return CUASR_STATUS_SUCCESS;
}

// Whether the elements of a strided box of bytes lie apart, seen from the smallest stride outwards; sufficient, and true
// of every view of a contiguous tensor.  *extent: bytes from the first to behind the last.
bool lies_apart(const int64_t (&stride)[4], const int64_t (&size)[4], int64_t bytes, int64_t* extent) {
  int order[4] = {0, 1, 2, 3};
  std::sort(order, order + 4, [&](int x, int y) { return stride[x] < stride[y]; });
  int64_t span = bytes;
  bool apart = true;
  for (int i : order) {
    if (size[i] <= 1) continue;
    apart = apart && stride[i] >= span;
    span += (size[i] - 1) * stride[i];
  }
  *extent = span;
  return apart;
}

int validate_reorder(const cuasr_b200_reorder_args_t* a) {
  if (a == nullptr) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (a->batch <= 0 || a->beams <= 0 || a->keep <= 0 || a->device < 0 || a->n_states < 0) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (a->n_states > CUASR_B200_REORDER_MAX_STATES || a->keep > 1024) return CUASR_STATUS_ERROR_NOT_SUPPORTED;
  if (a->parents == nullptr || a->ld_parents < a->keep || (a->n_states > 0 && a->states == nullptr))
    return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (!aligned(a->parents, 4) || !aligned(a->lengths, 4)) return CUASR_STATUS_ERROR_MISALIGNED_OPERAND;
  for (int i = 0; i < a->n_states; ++i) {
    const cuasr_b200_state_t& s = a->states[i];
    if (s.src == nullptr || s.dst == nullptr || s.bytes <= 0 || s.segments <= 0 || s.positions <= 0)
      return CUASR_STATUS_ERROR_INVALID_PROBLEM;
    if (s.ragged && a->lengths == nullptr) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
    const int64_t from[4] = {s.src_batch, s.src_beam, s.src_segment, s.src_position};
    const int64_t to[4] = {s.dst_batch, s.dst_beam, s.dst_segment, s.dst_position};
    const int64_t read[4] = {a->batch, a->beams, s.segments, s.positions}, written[4] = {a->batch, a->keep, s.segments, s.positions};
    for (int d = 0; d < 4; ++d)
      if (from[d] < 0 || to[d] < 0 || from[d] > INT64_MAX / 2 / std::max<int64_t>(1, read[d]) / 4 ||
          to[d] > INT64_MAX / 2 / std::max<int64_t>(1, written[d]) / 4)
        return CUASR_STATUS_ERROR_INVALID_PROBLEM;
    int64_t src_extent = 0, dst_extent = 0;
    const bool src_apart = lies_apart(from, read, s.bytes, &src_extent);
    if (!lies_apart(to, written, s.bytes, &dst_extent)) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
    if (s.src == s.dst && std::equal(from, from + 4, to)) {
      // rows that are only read must not be another search's that are written
      if (a->keep > a->beams || !src_apart) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
      if (a->keep > CUASR_B200_REORDER_MAX_IN_PLACE) return CUASR_STATUS_ERROR_NOT_SUPPORTED;
    } else {
      const char *x = static_cast<const char*>(s.src), *y = static_cast<const char*>(s.dst);
      if (x < y + dst_extent && y < x + src_extent) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
    }
    for (int j = 0; j < i; ++j)
      if (a->states[j].dst == s.dst || a->states[j].dst == s.src || a->states[j].src == s.dst) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  }
  return reorder_fits(*a) ? CUASR_STATUS_SUCCESS : CUASR_STATUS_ERROR_NOT_SUPPORTED;
}

// Runs `launch` on the device of the call.
template <typename Args, typename Launch>
int run_on_device(const Args& args, const char* kernel, Launch launch) {
  DeviceScope scope(args.device);
  if (!scope.ok()) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  DeviceInfo dev = {};
  if (!current_device_info(&dev)) return CUASR_STATUS_ERROR_INTERNAL;
  int launches = 0;
  const cudaError_t err = launch(args, dev, &launches);
  note_launches(kernel, launches);
  return err == cudaSuccess ? CUASR_STATUS_SUCCESS : CUASR_STATUS_ERROR_INTERNAL;
}

}  // namespace
}  // namespace cuasr_b200

using namespace cuasr_b200;

extern "C" {

int cuasr_b200_q4_product_can_implement(const cuasr_b200_q4_args_t* args) { return validate_q4(args); }

int cuasr_b200_q4_product(const cuasr_b200_q4_args_t* args) {
  const int st = validate_q4(args);
  return st != CUASR_STATUS_SUCCESS ? st : run_on_device(*args, "q4", launch_q4);
}

int cuasr_b200_beam_step_can_implement(const cuasr_b200_beam_args_t* args) { return validate_beam(args); }

size_t cuasr_b200_beam_step_workspace_size(const cuasr_b200_beam_args_t* args) {
  return validate_beam_sizes(args) == CUASR_STATUS_SUCCESS ? beam_workspace_bytes(*args) : 0;
}

int cuasr_b200_beam_step(const cuasr_b200_beam_args_t* args) {
  const int st = validate_beam(args);
  if (st != CUASR_STATUS_SUCCESS) return st;
  if (args->workspace == nullptr) return CUASR_STATUS_ERROR_WORKSPACE_NULL;
  if (args->workspace_bytes < beam_workspace_bytes(*args)) return CUASR_STATUS_ERROR_INVALID_PROBLEM;
  if (!aligned(args->workspace, 16)) return CUASR_STATUS_ERROR_MISALIGNED_OPERAND;
  return run_on_device(*args, "beam", launch_beam);
}

int cuasr_b200_reorder_states_can_implement(const cuasr_b200_reorder_args_t* args) { return validate_reorder(args); }

int cuasr_b200_reorder_states(const cuasr_b200_reorder_args_t* args) {
  const int st = validate_reorder(args);
  if (st != CUASR_STATUS_SUCCESS) return st;
  if (args->n_states == 0) return CUASR_STATUS_SUCCESS;
  return run_on_device(*args, "reorder", launch_reorder);
}

}  // extern "C"
