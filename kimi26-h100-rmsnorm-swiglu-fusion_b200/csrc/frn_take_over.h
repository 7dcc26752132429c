// frn_take_over.h -- which work a CTA does that takes over CTAs that have not been
// launched.  Apart from the kernel so that the rule can be run on the host.
#pragma once

#ifdef __CUDACC__
#define FRN_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FRN_HOST_DEVICE inline
#endif

namespace frn {

// The next number that has work: the CTA's own at first, then those of CTAs it
// takes over.  `hear` waits for the answer to the last request: false if no CTA
// was left.  `ask` makes the next request, which must not follow such an answer
// and must be answered before the CTA ends.  Answers come in no order that could
// be relied on, and a grid may have more numbers than there is work, so a number
// without work (`has_work`) says nothing about those still to come: only the end
// of the answers ends a CTA.  One request is under way after true, none after
// false.
template <typename Ask, typename Hear, typename HasWork>
FRN_HOST_DEVICE bool next_number(bool first, int own, Ask ask, Hear hear, HasWork has_work) {
  int number = own;
  for (bool got = first || hear(number); got; got = hear(number)) {
    ask();
    if (has_work(number)) return true;
  }
  return false;
}

}  // namespace frn
