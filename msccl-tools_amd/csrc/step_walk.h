// The steps of a product along its rows, of `k` values, `step` of them at a time: from step `first` to the last one, then those in
// front of it, each once.  Behind them nothing is left, so that copies that run ahead ask for nothing.
#ifndef MSCCLX_STEP_WALK_H
#define MSCCLX_STEP_WALK_H

namespace mscclx {

template <int STEP, int BYTES> struct StepWalk {  // BYTES: of a step
  int further, left;  // bytes from a row's first value to the step's, and the values from there on
  int turn, front;    // steps up to the turn, and those that come behind it
  constexpr explicit StepWalk(int k, int first = 0)
      : further((first - 1) * BYTES), left(k - (first - 1) * STEP), turn(first ? (k + STEP - 1) / STEP - first : -1), front(first) {}
  constexpr void next() {
    further += BYTES, left -= STEP;
    if (turn-- == 0) further = 0, left = front * STEP;  // whole steps: the partial one is the last of the row
  }
};

}  // namespace mscclx
#endif
