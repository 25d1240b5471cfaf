// capi_args.h -- what the entry points of the sequence and inference operators
// share: the plain form on the null stream, the _async form on the caller's, and
// checks of pointers.
#pragma once

#include <initializer_list>

#include "io_types.h"
#include "runtime.h"

namespace seera {

template <class F>
int now(F&& f) {
    clear_error();
    SEERA_TRY(f(nullptr));
    SEERA_HIP_TRY(hipDeviceSynchronize());
    note_device_synchronized();
    return SEERA_OK;
}
template <class F>
int later(void* stream, F&& f) {
    clear_error();
    SEERA_TRY(f(reinterpret_cast<hipStream_t>(stream)));
    note_async_work();
    return SEERA_OK;
}

inline int bad(const char* op, const char* what) { return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: %s", op, what); }

// Each of `ptrs` must not be null and must be aligned to a value of `bytes`.
inline int required(const char* op, size_t bytes, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs) {
        if (!p) return bad(op, "null device pointer");
        if (!aligned_to(p, bytes)) return bad(op, "a pointer is not aligned to its type");
    }
    return SEERA_OK;
}
// The same where a pointer is given.
inline int optional(const char* op, size_t bytes, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (!aligned_to(p, bytes)) return bad(op, "a pointer is not aligned to its type");
    return SEERA_OK;
}

}  // namespace seera
