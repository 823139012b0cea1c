// bindings.h -- what the translation units of the compiled binding astra_cuda._C share.
#pragma once

#include <torch/extension.h>

#include <string>

namespace astra_bind {

// Prints "Astra Fatal Error: ..." to stderr and throws, as AstraFatalError does
// (src/utils/astra_utils.cc:13-18).
[[noreturn]] void fatal(const std::string &msg);
// fatal(astra_last_error()) unless rc is ASTRA_OK.
void check(int rc);
// PyTorch's current HIP stream of a device.
void *stream_of(int device);

// The submodule astra_cuda._C.sequence (sequence_bindings.cpp).
void bind_sequence(pybind11::module_ &m);

}  // namespace astra_bind
