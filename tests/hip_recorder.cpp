// Stands in for the HIP runtime's calls of the library, so that a test without a GPU sees what a call
// would launch: every launch is written down, none runs, and memory is an address that nobody reads.
// A launch that HIP would refuse (2^32 threads or more along a dimension, more than 65535 workgroups along
// y or z) fails, and so does the one that `recorder_fail` names.  Load it before the library, globally.
#include <cstddef>
#include <cstdint>

struct dim3
{
    uint32_t x, y, z;
};
struct launch
{
    uint32_t grid[3], block[3];
    int32_t  failed;
};

static launch launches[4096];
static int    count = 0, fail_at = -1;

extern "C" {

int recorder_take(launch* to, int room)
{
    const int n = count < room ? count : room;
    for(int i = 0; i < n; ++i)
        to[i] = launches[i];
    const int all = count;
    count         = 0;
    fail_at       = -1;
    return all;
}
void recorder_fail(int which)
{
    fail_at = which;
}

int hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t, void*)
{
    const bool bad = uint64_t{grid.x} * block.x > 0xffffffffull || grid.y > 65535 || grid.z > 65535 || grid.x == 0
                     || grid.y == 0 || grid.z == 0 || count == fail_at;
    if(count < 4096)
        launches[count] = {{grid.x, grid.y, grid.z}, {block.x, block.y, block.z}, bad};
    ++count;
    return bad ? 1 : 0;
}
int hipGetDevice(int* device)
{
    *device = 0;
    return 0;
}
int hipDeviceGetAttribute(int* value, int, int)
{
    *value = 256;
    return 0;
}
int hipStreamIsCapturing(void*, int* status)
{
    *status = 0;
    return 0;
}
int hipMalloc(void** p, size_t)
{
    *p = reinterpret_cast<void*>(uintptr_t{1} << 40);
    return 0;
}
int hipGetSymbolAddress(void** p, const void*)
{
    *p = reinterpret_cast<void*>(uintptr_t{1} << 39);
    return 0;
}
int hipMemset(void*, int, size_t)
{
    return 0;
}
int hipFree(void*)
{
    return 0;
}
int hipDeviceSynchronize()
{
    return 0;
}
int hipGetLastError()
{
    return 0;
}
int hipEventCreateWithFlags(void** e, unsigned)
{
    *e = reinterpret_cast<void*>(uintptr_t{16});
    return 0;
}
int hipEventRecord(void*, void*)
{
    return 0;
}
int hipStreamWaitEvent(void*, void*, unsigned)
{
    return 0;
}
}
