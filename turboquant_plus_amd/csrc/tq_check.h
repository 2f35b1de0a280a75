// Argument checks shared by the files that hold C entry points.
#pragma once
#include "tq_internal.h"

#define REQUIRE(cond, code, ...)      \
    do {                              \
        if (!(cond)) {                \
            tq_set_error(__VA_ARGS__); \
            return code;              \
        }                             \
    } while (0)

static inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static inline bool fast_ok(const tq_handle *h) { return h->d == 128 && h->rotation == TQ_ROT_WHT && h->s1_32; }

static inline int check_fast(const tq_handle *h, const char *who) {
    REQUIRE(h, TQ_ERR_ARG, "%s: null handle", who);
    REQUIRE(fast_ok(h), TQ_ERR_UNSUPPORTED, "%s: needs d == 128 and WHT rotation (handle has d=%d, rotation=%d)", who,
            h->d, h->rotation);
    REQUIRE(h->bits >= 2 && h->bits <= 4, TQ_ERR_UNSUPPORTED, "%s: bits must be 2, 3 or 4 (got %d)", who, h->bits);
    return TQ_OK;
}
