// What the translation units of the C ABI share: the error text of the calling thread and the launch counter.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dnatok {

// Stores the text that dnatok_last_error() returns on this thread; returns `code`.
int abi_fail(int code, const char* fmt, ...);
void abi_count_launch();

}  // namespace dnatok
