// Host-side bookkeeping of the 8-bit layer operators, without a CUDA call of its own (the tests compile it without a GPU).
#pragma once
#include <atomic>
#include <cstdint>
#include <numeric>

namespace mmeb200 {

// How much of a kernel the device holds at once: `ask(&n)` puts the question when it first comes up (and is false where it fails),
// `known` keeps the answer. A failed question only rules out what needs the answer: `forget` clears the error that it left, and
// the result is `instead`, which is kept where it is a usable number (not negative: also for the answer "none"), else asked again.
template <typename Ask, typename Forget>
int device_holds(std::atomic<int>& known, Ask&& ask, Forget&& forget, int instead = -1) {
    int n = known.load(std::memory_order_relaxed);   // the answer + 1
    if (n) return n - 1;
    if (!ask(&n)) {
        forget();
        n = instead;
        if (n < 0) return n;
    } else if (n <= 0) {
        n = instead > 0 ? instead : 0;
    }
    known.store(n + 1, std::memory_order_relaxed);
    return n;
}

// Whether rows of `a_bytes` bytes at `a`, and of `b_bytes` at `b`, share no byte wherever they repeat: all strides of both (in
// bytes; those of dimensions with one element do not count) are multiples of one period, within which the rows lie apart. Column
// ranges of one matrix do.
template <typename Strides>
bool rows_lie_apart(uintptr_t a, uint64_t a_bytes, uintptr_t b, uint64_t b_bytes, const Strides& strides) {
    uint64_t period = 0;
    for (const uint64_t s : strides) period = std::gcd(period, s);
    if (period == 0) return false;
    const uint64_t behind = b >= a ? (b - a) % period : (period - (a - b) % period) % period;   // from a's row to the next of b
    return behind >= a_bytes && behind + b_bytes <= period;
}

// Marks the end of a call's use of shared memory on every way out of the call, errors in its middle included: work that was
// launched before them is still in flight. `mark()` returns a status.
template <typename Mark>
class UseMark {
    Mark mark;
    bool open = false;

public:
    explicit UseMark(Mark m) : mark(m) {}
    UseMark(const UseMark&) = delete;
    UseMark& operator=(const UseMark&) = delete;
    void begin() { open = true; }
    int end() {
        if (!open) return 0;
        open = false;
        return mark();
    }
    ~UseMark() { end(); }
};

}  // namespace mmeb200
