// Host-side launchers of the decoding operators: the kernels are compiled in the inst_*.cu files, decode.cu checks the
// arguments and plans the launches.  Also what decode.cu shares with abi.cu.
#pragma once

#include <atomic>

#include <cuda_runtime.h>

#include "../../include/cuasr_b200_decode.h"

namespace cuasr_b200 {

struct DeviceInfo {
  int sms;
  unsigned int* status;   // the device status word
};
// SM count and status word of the current device (abi.cu).
bool current_device_info(DeviceInfo* out);
// Adds to cuasr_b200_launch_count and names the call for cuasr_b200_last_kernel and cuasr_b200_last_route (abi.cu).
void note_launches(const char* kernel, int count);

// Opts a kernel in to `bytes` of dynamic shared memory (with its static more than 48 KB), once per device; `done` belongs
// to the kernel.
inline cudaError_t allow_shared_memory(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return err;
}

// Whether the sizes of valid arguments are within the kernel's.
bool q4_fits(const cuasr_b200_q4_args_t& args);
cudaError_t launch_q4(const cuasr_b200_q4_args_t& args, const DeviceInfo& dev, int* launches);

// Into how many parts the vocabulary of every prefix is cut; by the sizes alone, so that the workspace does not depend
// on the device.
int beam_parts(const cuasr_b200_beam_args_t& args);
size_t beam_workspace_bytes(const cuasr_b200_beam_args_t& args);
cudaError_t launch_beam(const cuasr_b200_beam_args_t& args, const DeviceInfo& dev, int* launches);

bool reorder_fits(const cuasr_b200_reorder_args_t& args);
cudaError_t launch_reorder(const cuasr_b200_reorder_args_t& args, const DeviceInfo& dev, int* launches);

}  // namespace cuasr_b200
