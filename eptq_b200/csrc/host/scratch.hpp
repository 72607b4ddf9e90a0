// What the files of the host extension share.
#pragma once

#include <torch/csrc/python_headers.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>

// The zero-filled scratch tensor of (device, stream), of at least so many bytes; only with the GIL held.
at::Tensor scratch_for(int device, const c10::cuda::CUDAStream& stream, size_t bytes);

// Functions of paged.cpp, ended by an empty entry.
extern PyMethodDef paged_methods[];
