// What the host sides of the library's operators share: launching a kernel, the scratch
// buffer of a device, alignment and the number of compute units.  The state behind them lives
// in gemm.hip.
#ifndef ROCM_WMMA_GEMM_HOST_SERVICES_HPP
#define ROCM_WMMA_GEMM_HOST_SERVICES_HPP

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <mutex>
#include <tuple>
#include <type_traits>
#include <utility>

#include "workspace_policy.hpp"

namespace rocm_wmma_gemm
{
namespace host
{

// Every kernel of the library is enqueued through this: the launch's own return code is kept
// per host thread, so that the entry points that return a status report what THEIR launches
// did, not an error some earlier call of anybody's left in the runtime's per-thread error
// state (hipPeekAtLastError cannot tell the two apart).
extern thread_local hipError_t launch_failure;

template<class... P, class... A, size_t... I>
void enqueue_impl(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, std::index_sequence<I...>,
                  A&&... a)
{
    std::tuple<std::remove_cv_t<std::remove_reference_t<P>>...> params(std::forward<A>(a)...);
    void*            ptrs[] = {static_cast<void*>(&std::get<I>(params))...};
    const hipError_t rc = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, ptrs, 0, stream);
    if(rc != hipSuccess && launch_failure == hipSuccess)
    {
        launch_failure = rc;
    }
}

template<class... P, class... A>
void enqueue(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, A&&... a)
{
    static_assert(sizeof...(P) == sizeof...(A), "one argument per kernel parameter");
    enqueue_impl(kernel, grid, block, stream, std::index_sequence_for<P...>{}, std::forward<A>(a)...);
}

// Library-owned scratch memory, one buffer per device: fp32 partial planes of split-K
// and zero-padded copies of ragged or misaligned operands.  Allocated on first use,
// grown when a call needs more (after a device-wide synchronisation, since kernels of
// earlier calls may still be reading the old buffer), never shrunk.  What a call may do
// with the buffer is decided by workspace_decide (workspace_policy.hpp).
constexpr size_t workspace_first_bytes = size_t{256} << 20;
constexpr size_t workspace_limit_bytes = size_t{16} << 30;
constexpr int    max_devices           = 64;
extern std::mutex workspace_mutex;
extern char* workspace_ptr[max_devices];
extern size_t workspace_size[max_devices];
// whether the buffer's address may sit in a captured graph: such a buffer is never freed
extern bool workspace_lent_to_capture[max_devices];
// The call that used the buffer last: its stream, and an event recorded behind its last
// kernel.
extern hipStream_t workspace_stream[max_devices];
extern hipEvent_t workspace_released[max_devices];
extern bool workspace_used[max_devices];

// One call's hold on the current device's buffer, from before its first kernel that
// touches the buffer is enqueued until after its last one is.  Calls that need the
// buffer are put in a queue on the device, whatever streams they are on: a call on
// another stream than the previous holder's makes its stream wait (on the device, the
// host never blocks) for the event recorded behind that holder's last kernel, so two
// streams may issue split-K or padded-copy GEMMs at the same time, from one host thread
// or several, as they may with the kernels that need no scratch memory.  A stream under
// graph capture is left out of this: it records and waits for nothing (the caller orders
// the replays of such a graph against other work that uses the buffer), it never
// allocates, frees or synchronises, and a buffer it was given stays allocated for good.
class workspace_lease
{
public:
    workspace_lease() = default;
    workspace_lease(const workspace_lease&)            = delete;
    workspace_lease& operator=(const workspace_lease&) = delete;

    // nullptr: no memory (or too much asked for, or the stream is capturing and the
    // buffer is not there yet or too small); the lease then holds nothing
    char* acquire(size_t bytes, hipStream_t stream)
    {
        if(bytes > workspace_limit_bytes || hipGetDevice(&dev_) != hipSuccess || dev_ < 0
           || dev_ >= max_devices)
        {
            return nullptr;
        }
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if(hipStreamIsCapturing(stream, &capture) != hipSuccess)
        {
            (void)hipGetLastError();
            capture = hipStreamCaptureStatusNone;
        }
        const bool capturing = capture != hipStreamCaptureStatusNone;
        lock_                = std::unique_lock<std::mutex>(workspace_mutex);
        const workspace_action action = workspace_decide(workspace_size[dev_], bytes, workspace_limit_bytes,
                                                         capturing, workspace_lent_to_capture[dev_]);
        if(action == workspace_action::refuse)
        {
            lock_.unlock();
            return nullptr;
        }
        if(action != workspace_action::use_existing)
        {
            if(action == workspace_action::grow_free_old)
            {
                (void)hipDeviceSynchronize();
                (void)hipFree(workspace_ptr[dev_]);
            }
            // (grow_retire_old: the old buffer stays allocated until the process ends,
            // for the graphs that hold its address)
            workspace_ptr[dev_]             = nullptr;
            workspace_size[dev_]            = 0;
            workspace_used[dev_]            = false;
            workspace_lent_to_capture[dev_] = false;
            const size_t want = workspace_grown_size(bytes, workspace_first_bytes);
            void*        p    = nullptr;
            if(hipMalloc(&p, want) != hipSuccess)
            {
                (void)hipGetLastError();
                lock_.unlock();
                return nullptr;
            }
            workspace_ptr[dev_]  = static_cast<char*>(p);
            workspace_size[dev_] = want;
        }
        stream_  = stream;
        ordered_ = !capturing;
        if(capturing)
        {
            workspace_lent_to_capture[dev_] = true;
        }
        if(ordered_ && workspace_released[dev_] == nullptr
           && hipEventCreateWithFlags(&workspace_released[dev_], hipEventDisableTiming) != hipSuccess)
        {
            (void)hipGetLastError();
            workspace_released[dev_] = nullptr;
            ordered_                 = false;
        }
        if(ordered_ && workspace_used[dev_] && workspace_stream[dev_] != stream)
        {
            (void)hipStreamWaitEvent(stream, workspace_released[dev_], 0);
        }
        held_ = true;
        return workspace_ptr[dev_];
    }

    ~workspace_lease()
    {
        if(held_ && ordered_)
        {
            (void)hipEventRecord(workspace_released[dev_], stream_);
            workspace_stream[dev_] = stream_;
            workspace_used[dev_]   = true;
        }
    }

private:
    std::unique_lock<std::mutex> lock_;
    hipStream_t                  stream_  = nullptr;
    int                          dev_     = 0;
    bool                         held_    = false;
    bool                         ordered_ = false;
};

// Counters of the workgroups that share a tile, and a tag for one launch that counts in them (see
// gemm.hip); nullptr without a device.  A caller holds the lease while its launches count.
constexpr size_t stream_arrival_slots = 4096;
unsigned int*    arrivals_of_current_device(bool noalloc);
unsigned int     next_arrival_epoch();

inline bool aligned16(const void* p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// CUs of the current device (cached per device), 0 if unknown.
inline size_t compute_units_of_current_device()
{
    static std::atomic<int> cached[64];
    int dev = 0;
    if(hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64)
    {
        return 0;
    }
    int cus = cached[dev].load(std::memory_order_relaxed);
    if(cus == 0)
    {
        if(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
        {
            return 0;
        }
        cached[dev].store(cus, std::memory_order_relaxed);
    }
    return static_cast<size_t>(cus);
}

} // namespace host
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_HOST_SERVICES_HPP
