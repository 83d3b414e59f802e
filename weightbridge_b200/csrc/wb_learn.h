// Registers the operators beside the sync (wb_learn.cpp) with the Python module.
#pragma once
#include <pybind11/pybind11.h>

namespace wb {
void bind_learn(pybind11::module_& m);
}
