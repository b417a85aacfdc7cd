// Where llmk_verify_drafts finds that a sequence ends, as it stands in the workspace between its
// launches. No device code: a program on the host may include it.
#pragma once

namespace llmk {
namespace verify {

// Logits over a temperature t, in log2 units.
struct Scale {
  double k;   // log2e / t
  float far;  // at a distance of -far and beyond weights are 0: about 10^9 / k
  int pad;
};

struct End {
  int first, end, row;  // its rows, and the one that gives its last token
  int last;             // that one stands behind all drafts
  int greedy, at;       // at: the row's argmax, where the choice is greedy
  float pm, qm;         // maxima of the target's and the draft model's row
  Scale by;
};
static_assert(sizeof(End) == 48, "workspace layout");

// z where its rows are the call's, else a sequence without rows. Rows become addresses, and the
// workspace is the caller's memory: where another stream's call or a temporary overwrites it
// between the launches, tokens are wrong, but nothing that is not the call's is read or written.
// s: the sequence; without row starts its row, and there are no drafts.
constexpr End checked(End z, int s, bool starts, int n_rows) {
  const bool rows = z.first >= 0 && z.end >= 0 && z.end <= n_rows &&
                    (starts || (z.first == s && z.end == s + 1));
  if (!rows || (z.end > z.first && (z.row < z.first || z.row >= z.end))) {
    z.first = z.end = 0;
  }
  if (z.end <= z.first) z.row = z.end - 1;
  z.last = z.row == z.end - 1;
  return z;
}

}  // namespace verify
}  // namespace llmk
