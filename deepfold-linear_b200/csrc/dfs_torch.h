// dfs_torch.h -- what the sources of the native torch extension share: errors,
// type codes and the device switch.
#pragma once

#include <torch/extension.h>

#include <cuda_runtime_api.h>
#include <stdexcept>
#include <string>

#include "dfsink.h"

namespace dfs_torch {

// Errors are thrown as std::runtime_error (pybind11 raises RuntimeError) with
// the message built here: a TORCH_CHECK whose message formats a number crashed
// the process in this torch build, inside any extension.
[[noreturn]] inline void fail(const std::string& msg) { throw std::runtime_error(msg); }
inline void require(bool ok, const char* msg) {
  if (!ok) fail(msg);
}

inline void check_rc(int rc, const char* what) {
  if (rc != DFS_OK)
    fail(std::string(what) + " failed: " + dfs_status_string(rc) + " (code " + std::to_string(rc) + ")");
}

inline int dtype_code(at::ScalarType t) {
  if (t == at::kBFloat16) return DFS_BF16;
  if (t == at::kHalf) return DFS_F16;
  return DFS_F32;
}

// Makes a device current for a scope and restores the previous one, with the
// plain runtime calls.
struct DeviceSwitch {
  int prev = -1;
  explicit DeviceSwitch(const at::Device& dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev.index()) cudaSetDevice(dev.index());
  }
  ~DeviceSwitch() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
  DeviceSwitch(const DeviceSwitch&) = delete;
  DeviceSwitch& operator=(const DeviceSwitch&) = delete;
};

// dfs_torch_attn.cpp: the local attention's functions.
void bind_window_attn(pybind11::module_& m);

}  // namespace dfs_torch
