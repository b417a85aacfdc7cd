// What the workers of llmk_kv8_attention note in the workspace for the launch that joins their
// parts. No device code: a program on the host may include it.
#pragma once

namespace llmk {
namespace kv8 {

// A unit that several workers share, as each of them notes it: one that began before the worker's
// share and one that ends behind it.
struct Shared {
  int first, last;      // the teams; first > last: there is none
  int column, columns;  // of the tile, from the sequence's first row on
  int row0, blind;      // the sequence's first row; columns in front of `blind` see nothing
  int pad[2];
};

// What the join reads becomes addresses, and the workspace is the caller's memory: where another
// stream's call or a temporary overwrites it between the launches, results are wrong, but nothing
// outside the workspace and the output is read or written. Two checks, so that the first waits for
// half a note only: the join by itself takes 4.9 us with them and 4.3 without at 48 sequences of up
// to 5 rows (5.3 with one check of all), the whole call 34.3 either way.
//
// Whether there is a unit of this team whose parts lie among those of `teams` teams with tiles of
// `most` columns.
constexpr bool is_unit(const Shared& o, int team, int teams, int most) {
  return o.first >= 0 && o.first <= team && team <= o.last && o.last < teams && o.columns > 0 &&
         o.columns <= most && o.column >= 0 && o.column <= 0x7FFF0000;
}
// The row of such a unit's column c < columns, -1 if it is none of the call's.
constexpr int row_of(const Shared& o, int c, int n_rows, int group) {
  const int row = (o.column + c) / group;
  return o.row0 >= 0 && row < n_rows - o.row0 ? o.row0 + row : -1;
}

}  // namespace kv8
}  // namespace llmk
