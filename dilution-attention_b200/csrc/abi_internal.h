// What the translation units of libdilution_b200.so share (host code).
#pragma once

#include <cuda_runtime.h>

namespace dil {

// Record an error for dilution_last_error() and return its code.
int abi_fail(int code, const char* fmt, ...);
// DILUTION_OK, or the error of the launch in front of it.
int abi_check_launch(const char* what);
// Accounts for one launch (and times it, where that is on) from its construction to its end.
class LaunchMark {
 public:
  LaunchMark(const char* name, cudaStream_t st);
  ~LaunchMark();
  LaunchMark(const LaunchMark&) = delete;
  LaunchMark& operator=(const LaunchMark&) = delete;

 private:
  void* prof_;
};
// The first bounded wait that ran out in a kernel of operators.cu (0: none), read and cleared.  Non-zero: could not be read.
int operators_read_status(int* code);

}  // namespace dil
