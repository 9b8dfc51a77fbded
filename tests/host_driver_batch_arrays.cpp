// The device arrays of a pool's batches and its counters as they are outgrown, over a stand-in for the
// device allocator that notes what was freed (host code only; test_host_batch_arrays.py).
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>

#include "device_pool.hpp"

namespace {
std::set<void*> live, freed;
int left = -1;  // allocations that still succeed (-1: all)
bool fills = true;
}  // namespace

extern "C" {
hipError_t hipMalloc(void** p, size_t n) {
    if (left == 0) return hipErrorOutOfMemory;
    if (left > 0) left--;
    *p = std::malloc(n);
    std::memset(*p, 0xAA, n);
    live.insert(*p);
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (p) {
        live.erase(p);
        freed.insert(p);  // (the memory stays: no address comes again)
    }
    return hipSuccess;
}
hipError_t hipMemset(void* p, int value, size_t n) {
    if (!fills) return hipErrorStreamCaptureUnsupported;
    std::memset(p, value, n);
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
}

#define CHECK(x)                                                     \
    do {                                                             \
        if (!(x)) {                                                  \
            std::printf("line %d: not so: %s\n", __LINE__, #x);      \
            return 1;                                                \
        }                                                            \
    } while (0)

int main() {
    {
        nitro::DecodeBatch d;
        d.reserve(512, 8);  // what a launch was captured over
        const int32_t *tables = d.tables.ptr, *pos = d.pos.ptr, *slots = d.slots.ptr;
        d.reserve(1024, 16);  // within the room there is
        CHECK(d.tables.ptr == tables && d.pos.ptr == pos && d.slots.ptr == slots);
        d.reserve(1088, 17);  // tables outgrown
        CHECK(d.tables.count >= 1088 && d.pos.count >= 17 && d.slots.count >= 17);
        // none of the old arrays was freed, and none is written for the new batch
        for (const int32_t* p : {tables, pos, slots}) {
            CHECK(live.count((void*)p) && !freed.count((void*)p));
            CHECK(p != d.tables.ptr && p != d.pos.ptr && p != d.slots.ptr);
        }
        const int32_t* now = d.tables.ptr;
        left = 1;  // the second of the three does not fit
        bool thrown = false;
        try {
            d.reserve(1 << 20, 1 << 16);
        } catch (const nitro::Error&) {
            thrown = true;
        }
        left = -1;
        CHECK(thrown && d.tables.ptr == now && d.tables.count < (1 << 20) && live.count((void*)now));
        d.reserve(1088, 17);
        CHECK(d.tables.ptr == now);
    }
    CHECK(live.empty());  // all of it goes with the batch
    {
        nitro::PrefillBatch p;
        p.reserve(512, 8, 192, 22, 20);
        const void* before[] = {p.tables.ptr, p.seqs.ptr, p.slots.ptr, p.row_pos.ptr, p.work.ptr, p.work_wide.ptr};
        p.reserve(1024, 16, 192, 38, 36);
        CHECK(p.tables.ptr == before[0] && p.work.ptr == before[4]);
        p.reserve(1088, 17, 192, 40, 38);
        const void* after[] = {p.tables.ptr, p.seqs.ptr, p.slots.ptr, p.row_pos.ptr, p.work.ptr, p.work_wide.ptr};
        for (int i = 0; i < 6; i++) {
            CHECK(live.count(const_cast<void*>(before[i])));
            CHECK(after[i] != before[i]);
        }
    }
    CHECK(live.empty());
    {
        // arrival counters: zeros from the first launch on, also after one whose fill failed
        nitro::KeptBuffer<int32_t> counters;
        fills = false;
        for (int i = 0; i < 2; i++) {
            bool thrown = false;
            try {
                counters.reserve(64, true);
            } catch (const nitro::Error&) {
                thrown = true;
            }
            CHECK(thrown && !counters.now.ptr);
        }
        fills = true;
        CHECK(counters.reserve(64, true) && !counters.reserve(64, true));
        for (size_t i = 0; i < counters.now.count; i++) CHECK(counters.now.ptr[i] == 0);
        int32_t* first = counters.now.ptr;
        first[3] = 7;
        fills = false;
        try {
            counters.reserve(1 << 20, true);
            CHECK(false);
        } catch (const nitro::Error&) {
        }
        CHECK(counters.now.ptr == first && counters.outgrown.empty());
        fills = true;
        CHECK(counters.reserve(1 << 20, true) && counters.now.ptr != first && live.count(first) && first[3] == 7);
        for (size_t i = 0; i < counters.now.count; i++) CHECK(counters.now.ptr[i] == 0);
    }
    CHECK(live.empty());
    std::printf("ok\n");
    return 0;
}
