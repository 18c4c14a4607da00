// What the C entry points of the policy's operators share: argument checks.
#pragma once
#include <hip/hip_runtime.h>

#include <climits>

#include "junqi_amd.h"
#include "jq_error.h"

namespace jq {

inline hipStream_t strm(void *s) { return reinterpret_cast<hipStream_t>(s); }

inline int check_dtype(int32_t dtype)
{
    if (dtype != JQ_F32 && dtype != JQ_BF16) return fail(JQ_E_ARG, "element type %d is neither JQ_F32 nor JQ_BF16", dtype);
    return JQ_OK;
}

inline size_t elem_bytes(int32_t dtype) { return dtype == JQ_F32 ? 4 : 2; }

inline bool aligned(const void *p, size_t to) { return (uintptr_t)p % to == 0; }

// A pointer to elements of `bytes`, or NULL.
inline int check_pointer(const void *p, size_t bytes, const char *name)
{
    if (!aligned(p, bytes)) return fail(JQ_E_ARG, "%s must be aligned to its element size", name);
    return JQ_OK;
}

inline int check_rows(const jq_rows &r, int32_t dtype, const char *name)
{
    if (!r.data) return fail(JQ_E_ARG, "null %s", name);
    if (!aligned(r.data, elem_bytes(dtype))) return fail(JQ_E_ARG, "%s must be aligned to its element size", name);
    return JQ_OK;
}

#define TRY(expr)                  \
    do {                           \
        const int rc_ = (expr);    \
        if (rc_) return rc_;       \
    } while (0)

}  // namespace jq
