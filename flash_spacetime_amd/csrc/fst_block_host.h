// What the two units of the host extension share.
#pragma once

#include <torch/extension.h>

#include "../../include/flash_spacetime.h"

// Entry points of layer norm and the feed-forward block (fst_block_host.cpp).
void bind_block_library(size_t norm_fwd, size_t norm_ws, size_t norm_bwd, size_t ffn_fwd, size_t ffn_ws,
                        size_t ffn_bwd, size_t last_error);
void define_block_operators(pybind11::module_& m);
