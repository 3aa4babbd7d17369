// TEST INFRASTRUCTURE: the layer operators' host-side bookkeeping (csrc/layer_host.h) with fakes of the CUDA calls behind it.
// Nothing in the product links or calls this file.
#include <vector>

#include "layer_host.h"

using namespace mmeb200;

extern "C" {
// Asks `times` times; the first `failures` questions fail, the others answer `answer`. results[i]: what came back; returns the
// number of questions put, and in *forgotten the number of errors cleared.
int hc_device_holds(int times, int failures, int answer, int instead, int* results, int* forgotten)
{
    std::atomic<int> known{0};
    int asked = 0;
    *forgotten = 0;
    for (int i = 0; i < times; i++)
        results[i] = device_holds(known, [&](int* n) { *n = answer; return ++asked > failures; }, [&] { ++*forgotten; }, instead);
    return asked;
}

int hc_rows_lie_apart(uint64_t a, uint64_t a_bytes, uint64_t b, uint64_t b_bytes, const uint64_t* strides, int n)
{
    return rows_lie_apart(uintptr_t(a), a_bytes, uintptr_t(b), b_bytes, std::vector<uint64_t>(strides, strides + n));
}

// A call that takes shared memory (or not), fails after its first launch (or not) and ends its use itself otherwise: how often
// the use was marked, and in *status what the call returned.
int hc_use_mark(int takes, int fails, int mark_status, int* status)
{
    int marks = 0;
    const auto mark = [&] { ++marks; return mark_status; };
    const auto call = [&]() -> int {
        UseMark<decltype(mark)> use(mark);
        if (takes) use.begin();
        if (fails) return -3;
        if (const int rc = use.end()) return rc;
        return 0;
    };
    *status = call();
    return marks;
}
}
