// Whether arrays of a call share memory (attn_check.hpp).  Plain C++, asked by the host and by
// CPU tests.
#pragma once

#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <utility>

namespace attn {

// Places that an array takes: the sums of stride * i, 0 <= i < count, over its axes, of which the
// first are the innermost.  `nested` where no two of them meet, and strides rise.
struct Axis {
    int64_t stride, count;
};
template <int N>
struct Box {
    Axis axes[N];
    bool nested = true;
    double reach[N + 1];  // places up to the last one of the inner axes; may pass 63 bits

    explicit Box(const Axis (&of)[N]) {
        for (int i = 0; i < N; ++i) axes[i] = {of[i].count > 1 ? of[i].stride : 0, of[i].count};
        for (int i = 1; i < N; ++i)
            for (int j = i; j > 0 && axes[j].stride < axes[j - 1].stride; --j) std::swap(axes[j], axes[j - 1]);
        reach[0] = 1;
        for (int i = 0; i < N; ++i) {
            nested = nested && (axes[i].count <= 1 || (double)axes[i].stride >= reach[i]);
            reach[i + 1] = reach[i] + (double)axes[i].stride * (double)(axes[i].count - 1);
        }
    }
    // Whether it has places in common with the same `apart` places on.  Of nested boxes.
    bool meets_itself(int64_t apart, int n = N) const {
        if (std::fabs((double)apart) >= reach[n]) return false;
        if (n == 0) return true;
        const Axis a = axes[n - 1];
        if (a.count <= 1) return meets_itself(apart, n - 1);
        int64_t i = apart / a.stride;  // steps of the axis: as many, or one more
        if (apart % a.stride < 0) --i;
        return (std::llabs(i) < a.count && meets_itself(apart - i * a.stride, n - 1)) ||
               (std::llabs(i + 1) < a.count && meets_itself(apart - (i + 1) * a.stride, n - 1));
    }
    // Whether it has places in [from, to).  Of boxes that are not nested, up to their last place.
    bool meets(int64_t from, int64_t to, int n = N) const {
        if (from >= to || to <= 0 || (double)from >= reach[n]) return false;
        if (n == 0 || !nested) return true;
        const Axis a = axes[n - 1];
        if (a.count <= 1) return meets(from, to, n - 1);
        // the last step of the axis that begins before `to`, and the one before it; what lies
        // between that one and `from` is passed whole
        int64_t i = (to - 1) / a.stride;
        if (i >= a.count) i = a.count - 1;
        if (meets(from - i * a.stride, to - i * a.stride, n - 1)) return true;
        return i > 0 && meets(from - (i - 1) * a.stride, to - (i - 1) * a.stride, n - 1);
    }
};

}  // namespace attn
