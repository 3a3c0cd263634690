// Between the two sources of the splat_host module (host_binding.cpp, paged_binding.cpp).
#pragma once

#include <Python.h>
#include <cstdint>

namespace splat_host {
PyMethodDef* paged_methods();              // paged_binding.cpp
// host_binding.cpp: the device's status word, and whether it exists and nothing has been reported through it
int32_t* status_word(int device);
bool status_ready(int device);
}  // namespace splat_host
