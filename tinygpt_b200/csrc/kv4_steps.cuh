// kv4_steps.cuh — which steps of 32 tokens the attention over the paged 4-bit cache goes over (kv4_attn.cu): plain arithmetic, for the device and the host alike.
// A step is looked up in the sequence's row of the table, so none may lie behind what the sequence has.
#pragma once

namespace b200 {

#ifdef __CUDACC__
#define B200_BOTH __host__ __device__ __forceinline__
#else
#define B200_BOTH inline
#endif

constexpr int kStep = 32;

struct Kv4Steps {
  int first, n;   // n: one at least, so that rows which see nothing are written, too
};
// Of a sequence whose rows stand from `pos` on and see tokens below `last` (0: none): from the step on that its first row sees under the window.  A window may lie
// behind all tokens: the last step then, whose tokens the mask drops.
B200_BOTH Kv4Steps kv4_seq_steps(int pos, int last, int window) {
  Kv4Steps s{0, 1};
  const int all = (last + kStep - 1) / kStep;
  if (window > 0 && pos >= window) {
    const int from = (pos - window + 1) / kStep, last_one = last > 0 ? (last - 1) / kStep : 0;
    s.first = from < last_one ? from : last_one;
  }
  if (all - s.first > 1) s.n = all - s.first;
  return s;
}
// How many of `many` steps from `step0` on a row at `high` sees some of (where there are tokens), and the first one that a row at `low` sees.
B200_BOTH int kv4_steps_end(int high, int last, int step0, int many) {
  const int upto = high / kStep + 1 - step0;
  return last <= 0 ? 0 : upto < many ? upto : many;
}
B200_BOTH int kv4_steps_begin(int low, int window, int step0) {
  const int from = window > 0 && low >= window ? (low - window + 1) / kStep - step0 : 0;
  return from > 0 ? from : 0;
}
// Of the sequence's steps those that rows at low … high see, counted from the sequence's first one; one at least.
B200_BOTH Kv4Steps kv4_rows_steps(int low, int high, int last, int window, const Kv4Steps& of) {
  const int end = last > 0 ? kv4_steps_end(high, last, of.first, of.n) : 1, begin = kv4_steps_begin(low, window, of.first), last_one = end > 1 ? end - 1 : 0;
  return {begin < last_one ? begin : last_one, end - begin > 1 ? end - begin : 1};
}

}  // namespace b200
