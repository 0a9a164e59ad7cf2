// Bindings of the bounded-cache operators (fd_stream_host.cpp) in the module
// of fd_hostpath.cpp.
#pragma once

#include <torch/extension.h>

void bind_stream_operators(py::module_& m);
