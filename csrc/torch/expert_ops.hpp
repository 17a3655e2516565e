#pragma once
#include <torch/python.h>

/** Adds the operators of dccl_b200/ops/experts.py to the extension module; 0, or -1 with a Python error set. */
int add_expert_ops(PyObject* module);
