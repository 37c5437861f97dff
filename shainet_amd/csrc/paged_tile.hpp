// How pages are read: the tiles of keys that the attention kernel takes, and which bytes of a row each lane asks for.  No device code, so
// that a host program can look at every head size.
#pragma once

namespace shainet {

constexpr int kPageF32 = 0, kPageBf16 = 1, kPageF16 = 2;
constexpr int page_element_bytes(int dtype) { return dtype == kPageF32 ? 4 : 2; }

// What is laid out how for pages of a type and heads of hd <= HD numbers, a multiple of 8.
template <int DTYPE, int HD>
struct PageTile {
  static constexpr int E = DTYPE == kPageF32 ? 4 : 2;      // bytes of a number
  static constexpr int S = DTYPE == kPageF32 ? 1 : 2;      // sixteens of keys of a tile
  static constexpr int KEYS = 16 * S;
  static constexpr int KEYS_EACH = 4 * S;                  // of a quarter of a wavefront
  static constexpr int CHUNKS = HD * E / 64;               // 16-byte pieces of a K row per lane
  static constexpr int PER = 16 / E;                       // numbers in one
  static constexpr int VEC = HD == 96 ? 3 * PER / 4 : HD / 16 < PER ? HD / 16 : PER;  // neighbouring columns of a V row per lane
  static constexpr int PIECES = HD / (16 * VEC);           // ... how often
  static constexpr int WORDS = VEC * E / 4;                // of 4 bytes, in one

  // Byte of a K row of `bytes` where the chunk u of quarter j begins; behind the row's end, where the query is 0, its first one again.
  static constexpr int key_byte(int u, int j, int bytes) {
    const int at = (u * 4 + j) * 16;
    return at < bytes ? at : 0;
  }
  // Whether a piece of a V row can begin in a row that ends before it does: 12 bytes of rows of 80 or 88 numbers.  (The others' divide
  // 8 numbers.)
  static constexpr bool RUNS_OVER = HD == 96;
  // The first column of lane m's piece u of a V row of hd numbers.  One that would run over the row's end ends with it instead, so that its
  // first columns are the piece before's last ones once more; where none runs over, one that begins behind the end is the first again.
  static constexpr int value_column(int u, int m, int hd) {
    const int d = VEC * (m + 16 * u);
    return RUNS_OVER ? (d < hd - VEC ? d : hd - VEC) : d < hd ? d : 0;
  }
};

}  // namespace shainet
