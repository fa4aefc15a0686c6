// The parts of the native bridge (one extension module).
#ifndef DEFORMOPS_AMD_BRIDGE_H_
#define DEFORMOPS_AMD_BRIDGE_H_

#include <pybind11/pybind11.h>

void define_operators(pybind11::module_& m);  // bridge_operators.cpp

#endif  // DEFORMOPS_AMD_BRIDGE_H_
