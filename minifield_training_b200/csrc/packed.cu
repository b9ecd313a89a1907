// Entry points with their arguments in one block.
//
// A foreign call through ctypes converts every argument by itself, 0.17 us
// each: 4.9 of the 11 us that a paged attention call of one token spent on the
// host, which is more than its kernels take. One packed block costs 1.1 us.
#include <string.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace mfb {
namespace packed {

// Slot 0 holds the flags, slot 1 + i argument i: a pointer, a signed 64-bit
// integer or a double. Integers outside their parameter's range are refused.
template <typename A>
A get(uint64_t slot, bool* ok) {
  if constexpr (std::is_pointer_v<A>) {
    return reinterpret_cast<A>(slot);
  } else if constexpr (std::is_floating_point_v<A>) {
    double d;
    memcpy(&d, &slot, sizeof(d));
    return (A)d;
  } else {
    *ok &= (uint64_t)(int64_t)(A)slot == slot;
    return (A)slot;
  }
}

template <typename... A, size_t... I>
int invoke(int (*f)(A...), const char* name, const uint64_t* slots, std::index_sequence<I...>) {
  MFB_CHECK_ARG(slots != nullptr, "%s: NULL arguments", name);
  bool ok = true;
  const std::tuple<A...> args{get<A>(slots[1 + I], &ok)...};
  MFB_CHECK_ARG(ok, "%s: an integer argument is out of range", name);
  if (slots[0] & MFB_PACKED_SHARED_WORKSPACE) {
    int capturing = 0;
    const int st = mfb_stream_is_capturing(std::get<sizeof...(A) - 1>(args), &capturing);
    if (st) return st;
    MFB_CHECK_ARG(!capturing, "%s: a captured call needs its own workspace (workspace=)", name);
  }
  return f(std::get<I>(args)...);
}

template <typename... A>
int call(int (*f)(A...), const char* name, const void* slots) {
  return invoke(f, name, static_cast<const uint64_t*>(slots), std::index_sequence_for<A...>{});
}

}  // namespace packed
}  // namespace mfb

#define MFB_PACKED(name) \
  extern "C" int name##_packed(const void* slots) { return mfb::packed::call(name, #name, slots); }

MFB_PACKED(mfb_qk_rotary_fwd)
MFB_PACKED(mfb_qk_rotary_bwd)
MFB_PACKED(mfb_paged_append)
MFB_PACKED(mfb_paged_attn)
MFB_PACKED(mfb_logits_process)
