// The table forms of the calls with many arguments: each word becomes the
// argument of its place.
#include <cstring>
#include <type_traits>
#include <utility>

#include "grs_common.cuh"

namespace grs {
namespace {

template <typename T>
T word_as(int64_t word) {
  if constexpr (std::is_pointer<T>::value) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(word));
  } else if constexpr (std::is_floating_point<T>::value) {
    double value;
    std::memcpy(&value, &word, sizeof(value));
    return static_cast<T>(value);
  } else {
    return static_cast<T>(word);
  }
}

template <typename... Args, size_t... I>
int call_words(int (*entry)(Args...), const int64_t* words, std::index_sequence<I...>) {
  return entry(word_as<Args>(words[I])...);
}
template <typename... Args>
int call_words(int (*entry)(Args...), const int64_t* words) {
  if (!words) return GRS_ERR_SHAPE;
  return call_words(entry, words, std::index_sequence_for<Args...>{});
}

}  // namespace
}  // namespace grs

extern "C" int grs_prompt_attention_words(const int64_t* words) {
  return grs::call_words(&grs_prompt_attention, words);
}
extern "C" int grs_shared_prefix_attention_words(const int64_t* words) {
  return grs::call_words(&grs_shared_prefix_attention, words);
}
extern "C" int grs_adjust_logits_words(const int64_t* words) {
  return grs::call_words(&grs_adjust_logits, words);
}
