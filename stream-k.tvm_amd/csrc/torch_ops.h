// What the units of libstreamk_torch.so share: the workspaces that the Python layer has told of (sk_torch_set_workspace).
#pragma once
#include <cstddef>
#include <shared_mutex>

namespace streamk_torch {

struct Buffer {
  void *ptr = nullptr;
  size_t bytes = 0;
};
// A call holds it, shared, from a look-up until its kernels are enqueued; a workspace is taken back under it, exclusively.
extern std::shared_mutex g_mutex;
// the workspace of a stream if there is one of that size (the caller holds g_mutex)
bool find_workspace(int device, void *stream, size_t bytes, Buffer *ws);

}  // namespace streamk_torch
