// How the C-ABI functions of the serving operators call theirs.
#pragma once

#include <string>

#include "common.hpp"

namespace tsm100 {

// Runs `op` with dev's CUDA device current; an exception (memory for a message) ends here.
template <typename F>
int32_t on_device(tsm100_device_t dev, F op) {
  const int32_t st = use_device(dev);
  if (st != TSM100_OK) return st;
  try {
    std::string err;
    const int32_t r = op(&err);
    if (r != TSM100_OK && !err.empty()) last_error_ref() = err;  // an operator called on the way has left its own
    return r;
  } catch (...) {
    return TSM100_ERR_RUNTIME;
  }
}

}  // namespace tsm100
