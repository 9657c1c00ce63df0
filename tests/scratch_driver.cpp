// DeviceBuffer::ensure over a HIP runtime made of counters: a block that a captured
// graph names stays where it is until its owner goes.
#include <cstdio>
#include <map>

#include "ra_internal.hpp"

namespace {
std::map<void*, size_t> allocated;  // live allocations
bool capturing = false, full = false;
uintptr_t next_address = 4096;
}  // namespace

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipDeviceSynchronize() { return capturing ? hipErrorStreamCaptureUnsupported : hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) {
    if (capturing) return hipErrorStreamCaptureUnsupported;
    if (full) return hipErrorOutOfMemory;
    *p = reinterpret_cast<void*>(next_address += 4096);
    allocated[*p] = n;
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (capturing) return hipErrorStreamCaptureUnsupported;
    allocated.erase(p);
    return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipMemcpy(void*, const void*, size_t, hipMemcpyKind) { return hipSuccess; }
}

#define CHECK(x)                                        \
    do {                                                \
        if (!(x)) {                                     \
            std::printf("line %d: %s\n", __LINE__, #x); \
            return 1;                                   \
        }                                               \
    } while (0)

int main() {
    using ra::DeviceBuffer;
    constexpr size_t kMiB = size_t(1) << 20;
    {  // Eager runs only: the smaller block is the next owner's.
        DeviceBuffer s, other;
        CHECK(s.ensure(kMiB, nullptr) == RA_OK);
        void* const first = s.get();
        CHECK(s.ensure(2 * kMiB, nullptr) == RA_OK && s.get() != first);
        CHECK(other.allocate(kMiB) == RA_OK && other.get() == first);
    }
    {  // A capture names the block: nobody else gets it, over any number of growths, until the owner goes.
        DeviceBuffer other;
        void *named, *again;
        {
            DeviceBuffer s;
            CHECK(s.ensure(3 * kMiB, nullptr) == RA_OK);
            named = s.get();
            capturing = true;
            CHECK(s.ensure(2 * kMiB, nullptr) == RA_OK && s.get() == named);
            capturing = false;
            CHECK(s.ensure(6 * kMiB, nullptr) == RA_OK && s.get() != named);
            CHECK(other.allocate(3 * kMiB) == RA_OK && other.get() != named);
            again = s.get();  // named by no graph yet
            capturing = true;
            CHECK(s.ensure(5 * kMiB, nullptr) == RA_OK && s.get() == again);
            capturing = false;
            CHECK(s.ensure(12 * kMiB, nullptr) == RA_OK);
            ra::pool_trim();
            CHECK(allocated.count(named) == 1 && allocated.count(again) == 1);
            // A growth that fails leaves the block and its size.
            capturing = true;
            CHECK(s.ensure(12 * kMiB, nullptr) == RA_OK);
            capturing = false;
            void* const last = s.get();
            const size_t bytes = s.bytes();
            full = true;
            CHECK(s.ensure(40 * kMiB, nullptr) == RA_ERR_OUT_OF_MEMORY);
            full = false;
            CHECK(s.get() == last && s.bytes() == bytes && allocated.count(last) == 1);
            // Moved with its owner.
            DeviceBuffer moved(std::move(s));
            CHECK(moved.get() == last && s.get() == nullptr && allocated.count(named) == 1);
            DeviceBuffer assigned;
            assigned = std::move(moved);
            CHECK(assigned.ensure(40 * kMiB, nullptr) == RA_OK && allocated.count(last) == 1);
        }
        ra::pool_trim();
        CHECK(allocated.count(named) == 0 && allocated.count(again) == 0 && allocated.size() == 1);  // other's
    }
    ra::pool_trim();
    CHECK(allocated.empty());
    std::printf("scratch ok\n");
    return 0;
}
