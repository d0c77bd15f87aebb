// Python bindings of the kernels around many samples of one prompt and a cache of bounded size (attention_groups.cu, decode_flat.cu, kv_evict.cu).
#pragma once
#include <pybind11/pybind11.h>

namespace nrl {
void bind_groups(pybind11::module_& m);
}
