// When the scales of w [N, K] travel in the product over 4-bit blocks on the bf16 matrix cores (f4_wide.h has the kernel).  Plain
// functions: a host program can walk them.
//
// A step is 64 of k, two scales of a row; they come for kScaleSteps steps at once, 16 bytes of a row, into two buffers in turn.  A slice
// of K may begin with an odd step, two bytes behind a word of four scales.  Rows are whole words, and loads give zeros past the end of
// the array by words: the first group begins with the word, an even step, so that no word of a load lies across the end (where the
// last step's scales of the last row would be lost, or bytes behind the array read).
#pragma once

namespace mx {
namespace f4 {

constexpr int kScaleSteps = 8;

// Of a slice that begins with step s0: the first step of its groups,
constexpr int scales_from(int s0) { return s0 & ~1; }
// the byte of a row where group t begins,
constexpr int scales_at(int s0, int t) { return 2 * (scales_from(s0) + kScaleSteps * t); }
// the group of step s, and the step's byte in it,
constexpr int scales_group(int s, int s0) { return (s - scales_from(s0)) / kScaleSteps; }
constexpr int scales_byte(int s, int s0) { return 2 * ((s - scales_from(s0)) % kScaleSteps); }
// and the group that is requested with the codes of step s, which come `buffers` - 1 steps ahead and begin behind the barrier of the
// step `buffers` before; 0 for none (group 0 goes before all codes).  Its buffer is free behind the barrier of the step 9 before
// its first, and it is needed behind the barrier of the step before its first, which waits for all that went with that first's codes.
constexpr int scales_with(int s, int s0, int buffers) {
  return s - scales_from(s0) + 1 >= buffers && (s - scales_from(s0) + 1 - buffers) % kScaleSteps == 0
             ? (s - scales_from(s0) + 1 - buffers) / kScaleSteps + 1
             : 0;
}

}  // namespace f4
}  // namespace mx
