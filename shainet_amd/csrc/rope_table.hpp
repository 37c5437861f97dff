// How long a table of cosines and sines becomes.  No device code, so that a host program can look at it.
#pragma once

namespace shainet {

// Of a table that is made longer than asked for; calls that do not know how far they will go ask for no more.
constexpr long long kMostTableBytes = 8LL << 30;
constexpr long long most_table_positions(int bytes_each) { return bytes_each > 0 ? kMostTableBytes / bytes_each : 0x7fffffffLL; }

// A table of `have` positions (0: none yet) is to have `positions` at least: doubled until it has, or as long as it may be, or as asked for if
// that is longer still.
constexpr int table_positions(int have, int positions, int bytes_each) {
  long long want = have > 0 ? have : 1024;
  while (want < positions) want *= 2;
  const long long most = most_table_positions(bytes_each) < 0x7fffffffLL ? most_table_positions(bytes_each) : 0x7fffffffLL;
  if (want > most) want = positions > most ? positions : most;
  return (int)want;
}

}  // namespace shainet
