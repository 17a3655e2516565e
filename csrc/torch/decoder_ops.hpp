#pragma once
#include <torch/python.h>

/** Adds the operators of dccl_b200/ops/decoder.py to the extension module; 0, or -1 with a Python error set. */
int add_decoder_ops(PyObject* module);
