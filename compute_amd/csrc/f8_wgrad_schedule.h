// Tiles of the weight gradient over 8-bit blocks and the order of a step's LDS traffic (f8_wgrad.hip has the kernel).
// Plain constants: a host program can walk them.
//
// A step of S tokens is kGroups groups of TK MFMAs, one operand of dy against the wave's TK operands of x.  LDS holds two
// steps: the present one's buffer is read while the next one's is filled, and the step's one barrier stands before its last
// kLast groups.  Every wave may run a whole step ahead of another but for that barrier, so
//   - all reads of the present buffer stand before it: behind it another wave may already be in the next step,
//     which fills that buffer again from its first group on;
//   - all writes into the next buffer stand before it, and all reads of that buffer behind it.
#pragma once

namespace mx {
namespace f8 {

// A workgroup computes kK (k) x kN (n) in WK x WN waves of 32 TK x 32 TN; P parts of dy (3: float32).
template <int WK_, int WN_, int TK_, int TN_, int S_, int P_, int OCC>
struct WGradTile {
  static constexpr int WK = WK_, WN = WN_, TK = TK_, TN = TN_, S = S_, P = P_, kThreads = 64 * WK * WN, kOccupancy = OCC;
  static constexpr int kK = 32 * TK * WK, kN = 32 * TN * WN, kPartBytes = 4 * kK * kN;

  static constexpr int kParts = S / 16, kPart = P * TN, kGroups = kParts * kPart;  // runs of 16 tokens, groups of a run
  static constexpr int kRing = 4, kLast = kRing - 1;  // slots of dy operands, groups behind the barrier
  static constexpr int kBarrier = kGroups - kLast;    // the barrier stands before this group

  // dy: the operand of group q is read kLast groups ahead; the first kLast of the next step behind the barrier.
  // x: the operands of the next run of 16 tokens are read in the first kXGroups groups of the present one, kXPer at a time: one a
  // group, unless the last run's would then come behind the barrier (with two groups a run).
  static constexpr int kXRoom = 2 * kPart - kLast;  // groups of the last run but one before the barrier
  static constexpr int kXGroups = TK < kXRoom ? TK : kXRoom, kXPer = (TK + kXGroups - 1) / kXGroups;
  // The next step's first run of x, behind the barrier: kNextPer in each of its last kNextGroups groups.
  static constexpr int kNextGroups = kLast < kPart ? kLast : kPart, kNextPer = (TK + kNextGroups - 1) / kNextGroups;
  // Staging of the next step: kPieces pieces, half a chunk of x or one of dy, mixed evenly, in the groups from kStageFrom.
  static constexpr int kXChunks = S * kK / 16 / kThreads, kDChunks = S * kN / 8 / kThreads;  // of a thread
  static constexpr int kPieces = 2 * kXChunks + kDChunks;
  static constexpr int kStageGroups = kBarrier < kPieces ? kBarrier : kPieces, kStageFrom = kBarrier - kStageGroups;
  static constexpr int kPerGroup = (kPieces + kStageGroups - 1) / kStageGroups;

  static_assert(kParts % 2 == 0 && kPart >= TK, "the sets of x operands alternate, and one is read while the other is used");
  static_assert(kGroups % kRing == 0, "the ring's slots are the same in every step");
  static_assert(kXRoom >= 1 && (kParts - 2) * kPart + kXGroups <= kBarrier, "the last x operands of a step are read before its barrier");
  static_assert(kXGroups * kXPer >= TK && kXGroups <= kPart && kNextGroups * kNextPer >= TK, "all operands are read");
  static_assert(kXChunks * 16 * kThreads == S * kK && kDChunks * 8 * kThreads == S * kN, "whole chunks");
};

using WGradTile256 = WGradTile<4, 2, 2, 4, 64, 1, 2>;
using WGradTile128 = WGradTile<2, 2, 2, 2, 64, 1, 2>;
using WGradTile256F32 = WGradTile<4, 2, 2, 4, 32, 3, 2>;  // steps of 32 tokens: LDS holds dy three times
using WGradTile128F32 = WGradTile<2, 2, 2, 2, 32, 3, 2>;

}  // namespace f8
}  // namespace mx
