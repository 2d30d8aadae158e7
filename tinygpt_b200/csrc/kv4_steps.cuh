// kv4_steps.cuh — which steps of 32 tokens the attention over the paged 4-bit cache goes over, and how the line of all of them is cut (kv4_attn.cu): plain arithmetic, for
// the device and the host alike.  A step is looked up in the sequence's row of the table, so none may lie behind what the sequence has; and every search ends
// whatever it is asked for.
#pragma once

namespace b200 {

#ifdef __CUDACC__
#define B200_BOTH __host__ __device__ __forceinline__
#else
#define B200_BOTH inline
#endif

constexpr int kStep = 32;
constexpr int kAhead = 2;     // steps that an item costs before its first token
constexpr int kGrid = 148;    // CTAs

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

// How the line is cut: `warps` pieces, `each` CTA having so many of them; piece w starts at about line·w / warps (as fp32 has it: the same for everyone).  A piece is no shorter than a step and what
// comes before it, and short lines are spread over the CTAs first.
struct Kv4Cut {
  int line, warps, each, whole, rest;   // line = whole·warps + rest
  float inverse;
  B200_BOTH Kv4Cut(int line_, int most) : line(line_) {
    const int pieces = line / (kAhead + 1);
    warps = pieces < 1 ? 1 : pieces < kGrid * most ? pieces : kGrid * most;
    each = (warps + kGrid - 1) / kGrid;
#ifdef __CUDA_ARCH__
    inverse = __frcp_rn((float)warps);
#else
    inverse = 1.f / (float)warps;
#endif
    whole = line / warps;
    rest = line - whole * warps;
  }
  B200_BOTH int start(int w) const { return w < warps ? w * whole + (int)((float)(w * rest) * inverse) : line; }
  B200_BOTH int owner(int x) const {   // whose piece x is; of a place off the line its nearest piece's
    int v = (int)((float)x / (float)(line > 0 ? line : 1) * (float)warps);
    v = v < 0 ? 0 : v > warps - 1 ? warps - 1 : v;
    while (v > 0 && start(v) > x) --v;
    while (v < warps - 1 && start(v + 1) <= x) ++v;
    return v;
  }
};
// The item at place `at` of a line, of those that begin at `base` and have `steps` each: the how manieth; its steps lie at begin … end − 1.  `limit`: where the line of its sequence
// ends (behind `at`), which an item does not pass, so that who goes on at its end gets on, and stays on the line, also if `steps` is not what the line was made of.
struct Kv4Item {
  int number, begin, end;
};
B200_BOTH Kv4Item kv4_item(int at, int base, int limit, int steps) {
  const unsigned length = (unsigned)(steps + kAhead), off = (unsigned)(at - base);
#ifdef __CUDA_ARCH__
  unsigned number = (unsigned)((float)off * __frcp_rn((float)length));   // (a division costs more than these)
#else
  unsigned number = (unsigned)((float)off * (1.f / (float)length));
#endif
  while (number * length > off) --number;
  while ((number + 1) * length <= off) ++number;
  const int begin = base + (int)(number * length) + kAhead;
  return {(int)number, begin, steps < limit - begin ? begin + steps : limit};
}
// The pieces that hold an item which `from`, of CTA `cta`, does not finish: from … to, of which CTAs in0 … in1 − 1 leave one part each (none: in0 >= in1).
struct Kv4Pieces {
  int from, to, in0, in1, each;   // from < 0: none
  int before, whole, parts;       // parts of pieces in front of those CTAs, of the CTAs, of all
  B200_BOTH int piece(int k) const { return k < before ? from + k : k < before + whole ? (in0 + k - before) * each : in1 * each + k - before - whole; }
};
B200_BOTH Kv4Pieces kv4_pieces(const Kv4Cut& cut, int cta, int me, int begin, int end) {
  Kv4Pieces p;
  p.from = me;
  p.to = cut.owner(end - 1);
  if (p.to < me) p.to = me;
  p.in0 = cut.start(cta * cut.each) == begin ? cta : cta + 1;
  p.in1 = cut.start(p.to + 1) == end && (p.to + 1) % cut.each == 0 ? (p.to + 1) / cut.each : p.to / cut.each;
  if (cut.each == 1) p.in1 = p.in0;
  p.each = cut.each;
  const bool some = p.in0 < p.in1;
  p.before = some ? p.in0 * p.each - me : p.to - me + 1;
  p.whole = some ? p.in1 - p.in0 : 0;
  p.parts = p.before + p.whole + (some ? p.to - p.in1 * p.each + 1 : 0);
  return p;
}
// whether a CTA's pieces are all of this item alone, so that its warps leave one part
B200_BOTH bool kv4_inside(const Kv4Cut& cut, int cta, int begin, int end) {
  return cut.each > 1 && cut.start(cta * cut.each) >= begin && cut.start((cta + 1) * cut.each) <= end && (cta + 1) * cut.each <= cut.warps;
}

}  // namespace b200
