// What the binding's translation units share.
#pragma once
#include <torch/extension.h>

torch::Tensor status_word(const torch::Tensor& like);   // binding.cpp
void bind_paged(pybind11::module& m);                   // binding_paged.cpp
