// What the C entry points of level 1 share (tensor_api.cpp, decode_api.cpp): the handle behind wkf_tensor, the per-device
// settings, and the mapping of exceptions to status codes.
#pragma once

#include <new>
#include <string>
#include <utility>
#include <vector>

#include "graph.h"

// hip_ffi.cpp owns the thread-local error string; this hook lets the upper layers set it.
void wkf_set_last_error_(const char* msg);

struct wkf_tensor {
  wkf_device* dev;
  wkf::NodeP node;
  std::vector<wkf::LaunchRecord> launches;  // of the last materialize
};

namespace wkf {

// The settings of `dev` (tuning knobs are read from the environment on first use).
Settings settings_for(wkf_device* dev);

// Runs `f`, mapping exceptions to status codes + wkf_last_error().
template <typename F>
int guarded(F&& f) {
  try {
    f();
    return WKF_OK;
  } catch (const Error& e) {
    wkf_set_last_error_(e.what());
    return e.code;
  } catch (const std::bad_alloc&) {
    wkf_set_last_error_("host allocation failed");
    return WKF_ERR_OOM;
  } catch (const std::exception& e) {
    wkf_set_last_error_(e.what());
    return WKF_ERR_INVALID_ARG;
  } catch (...) {
    wkf_set_last_error_("unknown exception");
    return WKF_ERR_INVALID_ARG;
  }
}

inline wkf_tensor* wrap(wkf_device* dev, NodeP n) {
  wkf_tensor* t = new wkf_tensor();
  t->dev = dev;
  t->node = std::move(n);
  return t;
}

inline void need(const void* p, const char* what) {
  if (!p) invalid(std::string(what) + ": null argument");
}

inline NodeP make(NodeKind k, DType dt, std::vector<size_t> shape) {
  NodeP n = std::make_shared<Node>();
  n->kind = k;
  n->dtype = dt;
  n->shape = std::move(shape);
  return n;
}

}  // namespace wkf
