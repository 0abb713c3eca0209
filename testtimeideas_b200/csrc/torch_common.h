// What the operator files of libttt_torch.so share (defined in torch_ops.cpp):
// the per-device error word with its host mirror, and the status check.
#pragma once

#include <ATen/ATen.h>

namespace ttt_torch {

// The device's error word (int32 [1]), created on first use; the device must be current.
at::Tensor error_word_for(int dev);
// Raises (and clears both words) if a kernel has reported an error to the host mirror.
void raise_if_pending(int dev, at::Tensor& word);
// Raises with the library's description of a status other than TTT_OK.
void check(int status, const char* op);

}  // namespace ttt_torch
