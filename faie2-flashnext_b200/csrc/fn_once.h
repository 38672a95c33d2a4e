// What has been done once for a kernel on a device: a kernel's attributes belong to the device that was current, and entries may be
// called from several threads.
#pragma once

#include <mutex>
#include <set>
#include <utility>

namespace fn {

class OncePerDevice {
    std::mutex m;
    std::set<std::pair<const void *, int>> done;

public:
    bool has(const void *kernel, int device) {
        const std::lock_guard<std::mutex> lock(m);
        return done.count({kernel, device}) != 0;
    }
    void add(const void *kernel, int device) {
        const std::lock_guard<std::mutex> lock(m);
        done.insert({kernel, device});
    }
};

}  // namespace fn
