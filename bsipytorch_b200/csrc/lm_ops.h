// Functions that lm_ops.cpp adds to the `bsi_ops` module.
#pragma once

#include <pybind11/pybind11.h>

void register_lm_ops(pybind11::module& m);
