// The profiling hook (ttt_attn_profile_enable) for entry points outside capi.cu:
// brackets what is launched on `stream` during the span's life with two events
// while profiling is on.
#pragma once

#include <cuda_runtime.h>

namespace ttt {

void* prof_begin(int kind, cudaStream_t stream);  // null while profiling is off
void prof_end(void* span);

class ProfSpan {
 public:
  ProfSpan(int kind, void* stream) : span_(prof_begin(kind, static_cast<cudaStream_t>(stream))) {}
  ~ProfSpan() {
    if (span_ != nullptr) prof_end(span_);
  }
  ProfSpan(const ProfSpan&) = delete;
  ProfSpan& operator=(const ProfSpan&) = delete;

 private:
  void* span_;
};

}  // namespace ttt
