// s1_call: the calls of a decoding step with their arguments as an array of words. A foreign-function layer that converts argument
// by argument (Python's ctypes: 0.2 us each) spends longer on the 27 arguments of s1_attention_paged than the kernel on a short context.
#include <stdint.h>
#include <string.h>

#include <limits>
#include <tuple>
#include <type_traits>
#include <utility>

#include "context.h"

namespace {

template <typename T>
T from_word(int64_t w, bool& ok) {
    if constexpr (std::is_pointer_v<T>) {
        return reinterpret_cast<T>(static_cast<uintptr_t>(w));
    } else if constexpr (std::is_floating_point_v<T>) {
        double d;
        memcpy(&d, &w, sizeof(d));
        return static_cast<T>(d);
    } else {
        if (sizeof(T) < sizeof(w) && (w < static_cast<int64_t>(std::numeric_limits<T>::min()) || w > static_cast<int64_t>(std::numeric_limits<T>::max()))) ok = false;
        return static_cast<T>(w);
    }
}

template <typename... A, size_t... I>
int apply(s1_ctx* ctx, const char* who, int (*f)(s1_ctx*, A...), const unsigned char* args, int words, std::index_sequence<I...>) {
    if (words != static_cast<int>(sizeof...(A))) return s1_fail(ctx, S1_EINVAL, "%s: %d argument words, not %d", who, static_cast<int>(sizeof...(A)), words);
    int64_t w[sizeof...(A)];
    memcpy(w, args, sizeof(w));  // (the array may lie anywhere)
    bool ok = true;
    const std::tuple<A...> a{from_word<A>(w[I], ok)...};
    if (!ok) return s1_fail(ctx, S1_EINVAL, "%s: an int argument is beyond 32 bits", who);
    return f(ctx, std::get<I>(a)...);
}

template <typename... A>
int apply(s1_ctx* ctx, const char* who, int (*f)(s1_ctx*, A...), const void* args, int words) {
    return apply(ctx, who, f, static_cast<const unsigned char*>(args), words, std::index_sequence_for<A...>{});
}

}  // namespace

extern "C" int s1_call(s1_ctx* ctx, int which, const void* args, int words) {
    if (!ctx) return S1_EINVAL;
    if (!args) return s1_fail(ctx, S1_EINVAL, "s1_call: null pointer");
    switch (which) {
        case S1_CALL_BLOCK_TABLES: return apply(ctx, "s1_block_tables", s1_block_tables, args, words);
        case S1_CALL_CACHE_WRITE: return apply(ctx, "s1_cache_write", s1_cache_write, args, words);
        case S1_CALL_ATTENTION_PAGED: return apply(ctx, "s1_attention_paged", s1_attention_paged, args, words);
        case S1_CALL_GATED_DELTA_RULE_STEP: return apply(ctx, "s1_gated_delta_rule_step", s1_gated_delta_rule_step, args, words);
        default: return s1_fail(ctx, S1_EINVAL, "s1_call: no call %d", which);
    }
}
