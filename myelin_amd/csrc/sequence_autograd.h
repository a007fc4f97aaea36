// Adds the sequence-model operators of sequence_autograd.cpp to the extension
// module.
#pragma once

#include <torch/extension.h>

void register_sequence_operators(pybind11::module_ &m);
