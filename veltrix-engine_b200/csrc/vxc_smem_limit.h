// vxc_smem_limit.h — the dynamic shared memory that kernels may be launched
// with, raised as calls need it.  (Plain C++: Api is the CUDA runtime, or a
// stand-in for it in a test.)
#pragma once
#include <pthread.h>
#include <stddef.h>

#include <atomic>

#define VXC_SMEM_DEFAULT (48 * 1024)   // allowed without asking

// The limit is per kernel and device and only ever raised.  A kernel that has
// it on a device is remembered, since asking costs a launch's time.  Reading,
// setting and remembering happen under one lock: two threads that read the same
// limit and set different ones could leave the smaller.
// Api: error, ok (its value of success), device(int *), limit(const void *, size_t *),
// set_limit(const void *, size_t).
template <class Api>
typename Api::error vxc_smem_allow(const void *kernel, size_t bytes) {
    if (bytes <= VXC_SMEM_DEFAULT) return Api::ok;
    struct Entry {
        std::atomic<const void *> kernel;
        std::atomic<size_t> bytes[64];
    };
    static Entry seen[64];
    static pthread_mutex_t lock = PTHREAD_MUTEX_INITIALIZER;
    int dev = 0;
    typename Api::error e = Api::device(&dev);
    if (e != Api::ok) return e;
    Entry *own = nullptr;
    for (Entry &s : seen) {
        const void *k = s.kernel.load(std::memory_order_acquire);
        if (!k && s.kernel.compare_exchange_strong(k, kernel)) k = kernel;
        if (k == kernel) {
            own = &s;
            break;
        }
    }
    if (own && dev < 64 && own->bytes[dev].load(std::memory_order_acquire) >= bytes) return Api::ok;
    pthread_mutex_lock(&lock);
    size_t have = 0;
    e = Api::limit(kernel, &have);
    if (e == Api::ok && have < bytes) {
        e = Api::set_limit(kernel, bytes);
        have = bytes;
    }
    if (e == Api::ok && own && dev < 64) own->bytes[dev].store(have, std::memory_order_release);
    pthread_mutex_unlock(&lock);
    return e;
}
