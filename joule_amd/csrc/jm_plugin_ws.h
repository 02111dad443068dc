// Workspace policy of the calls without a store (the plugin products, the 4-bit
// cache's attention, sampling), host code only (the CPU tests compile it on its
// own).  Each (device, stream) keeps one persistent buffer, and a call either
// reuses it, grows it, or (under stream capture) takes a stream-ordered
// allocation that it frees after its kernels:
//   - a call holds its buffer until all its kernels are enqueued: of two host
//     threads on one stream the second's kernels come behind the first's, not
//     between them, where they would overwrite what one kernel hands to the next;
//   - a graph being captured must not bake in the persistent buffer: a later
//     eager call on the stream that needs more space would replace it while
//     the graph still points at it;
//   - a grown buffer's predecessor is retired, not freed: kernels that are
//     enqueued may still use it, and freeing would wait for them.  Retired
//     buffers live until the process ends; with the growth below they total at
//     most the final size.
#pragma once

#include <stddef.h>

#include <list>
#include <mutex>
#include <vector>

namespace jm {

// The persistent buffer of one (device, stream); p, bytes and retired belong to
// who holds mu.
struct PluginBuf {
    PluginBuf(int d, void* s) : dev(d), st(s) {}
    const int dev;
    void* const st;
    std::mutex mu;
    void* p = nullptr;
    size_t bytes = 0;
    std::vector<void*> retired;             // replaced buffers, kept until the process ends
};

class PluginBufs {
  public:
    // The buffer of (dev, st), which lives as long as this; made at its first use.
    PluginBuf& of(int dev, void* st) {
        std::lock_guard<std::mutex> lk(mu_);
        for (PluginBuf& b : bufs_)
            if (b.dev == dev && b.st == st) return b;
        bufs_.emplace_back(dev, st);
        return bufs_.back();
    }

  private:
    std::mutex mu_;
    std::list<PluginBuf> bufs_;             // (entries stay where they are)
};

// Workspace of one call.  As long as it lives no other call takes the buffer.
struct PluginWs {
    void* p = nullptr;
    bool async = false;                     // p is the call's own, to be freed after its kernels
    std::unique_lock<std::mutex> held;
};

enum class WsAction { Reuse, StreamOrdered, Grow };

inline WsAction plugin_ws_action(size_t have_bytes, size_t need, bool capturing) {
    if (capturing) return WsAction::StreamOrdered;
    if (have_bytes >= need) return WsAction::Reuse;
    return WsAction::Grow;
}

// bytes to allocate when growing: at least 1 MiB and at least twice the
// buffer it replaces, so that a stream's retired buffers sum to less than
// its current one
inline size_t plugin_ws_grow(size_t have_bytes, size_t need) {
    size_t g = need > ((size_t)1 << 20) ? need : ((size_t)1 << 20);
    if (g < 2 * have_bytes) g = 2 * have_bytes;
    return g;
}

}  // namespace jm
