// The operators' entry points with their arguments as one array of words: a foreign caller pays for every argument it converts
// (37 of them: 6 us in ctypes, packed 1.6), which is a third of a single token's call.
#include <string.h>
#include <tuple>
#include <type_traits>
#include <utility>

#include "blk_common.h"

namespace ndb {

template <typename A>
static A word(int64_t w, bool& fits) {
    if constexpr (std::is_pointer<A>::value) {
        return reinterpret_cast<A>(static_cast<uintptr_t>(w));
    } else if constexpr (std::is_same<A, float>::value) {
        double d;
        memcpy(&d, &w, sizeof d);
        return (float)d;
    } else {
        if (w != (int64_t)(A)w) fits = false;
        return (A)w;
    }
}

template <typename... A, size_t... I>
static int unpack(int (*fn)(A...), const int64_t* words, nd_stream_t stream, std::index_sequence<I...>) {
    bool fits = true;
    using All = std::tuple<A...>;
    const std::tuple<std::tuple_element_t<I, All>...> args{word<std::tuple_element_t<I, All>>(words[I], fits)...};
    NDB_REQUIRE(fits, "nd_block_packed", "an argument does not fit its type");
    return fn(std::get<I>(args)..., stream);
}

template <typename... A>
static int packed(int (*fn)(A...), const int64_t* words, int count, nd_stream_t stream) {
    NDB_REQUIRE(words && count == (int)sizeof...(A) - 1, "nd_block_packed", "wrong number of arguments");
    return unpack(fn, words, stream, std::make_index_sequence<sizeof...(A) - 1>{});
}

}  // namespace ndb

using namespace ndb;

extern "C" int nd_block_packed(int call, const int64_t* words, int count, nd_stream_t stream) {
    switch (call) {
        case ND_CALL_QK_NORM_ROPE: return packed(nd_qk_norm_rope, words, count, stream);
        case ND_CALL_QK_NORM_ROPE_BWD: return packed(nd_qk_norm_rope_bwd, words, count, stream);
        case ND_CALL_DIFF_ATTENTION: return packed(nd_diff_attention, words, count, stream);
        case ND_CALL_DIFF_ATTENTION_BWD: return packed(nd_diff_attention_bwd, words, count, stream);
        case ND_CALL_GATED_FFN: return packed(nd_gated_ffn, words, count, stream);
        case ND_CALL_GATED_FFN_BWD: return packed(nd_gated_ffn_bwd, words, count, stream);
        default: return fail_arg("nd_block_packed", "unknown call");
    }
}
