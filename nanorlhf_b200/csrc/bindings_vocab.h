// Python bindings of the kernels over rows of logits (top_logits.cu, distill.cu, sample_filtered.cu).
#pragma once
#include <pybind11/pybind11.h>

namespace nrl {
void bind_vocab(pybind11::module_& m);
}
