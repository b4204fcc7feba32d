// launch_lock.h -- keeps the launches of one call together on the stream.
//
// A call of several kernels hands its scratch from one to the next.  Two host threads that call on the same stream with
// the same scratch may otherwise put kernel A1, B1, A2, B2 on it, and A2 reads what B1 left.  Locks are shared by scratch
// address, so calls with scratch of their own rarely meet.
#pragma once
#include <pthread.h>
#include <stdint.h>

namespace mq {

class LaunchLock {
public:
    explicit LaunchLock(const void* scratch) : m_(lock_of(scratch)) { pthread_mutex_lock(m_); }
    ~LaunchLock() { pthread_mutex_unlock(m_); }
    LaunchLock(const LaunchLock&) = delete;
    LaunchLock& operator=(const LaunchLock&) = delete;

private:
    static pthread_mutex_t* lock_of(const void* scratch) {
        static pthread_mutex_t locks[8] = {PTHREAD_MUTEX_INITIALIZER, PTHREAD_MUTEX_INITIALIZER, PTHREAD_MUTEX_INITIALIZER,
                                           PTHREAD_MUTEX_INITIALIZER, PTHREAD_MUTEX_INITIALIZER, PTHREAD_MUTEX_INITIALIZER,
                                           PTHREAD_MUTEX_INITIALIZER, PTHREAD_MUTEX_INITIALIZER};
        return &locks[((uintptr_t)scratch >> 9) & 7u];   // torch's allocations are multiples of 512 bytes
    }
    pthread_mutex_t* m_;
};

}  // namespace mq
