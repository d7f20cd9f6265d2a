// beam.h -- beam search's selection step.  No reference counterpart (the reference has no generation loop).
#pragma once

#include "inferno/core/tensor.h"

namespace Inferno {

struct BeamStep {
    Tensor tokens, parents;  // Int32 [groups, beams]: the next token, the beam of the group that it continues
    Tensor scores;           // Float32 [groups, beams], best first
    Tensor finished;         // Int32 [groups, beams]; undefined where eos < 0
};

// The best `beams` (at most 32) of every group's beams x V continuations by score + log-softmax(logits), on a
// HIP device: logits [groups * beams, V] or [groups * beams, 1, V] with dense rows, scores Float32 and finished
// Int32 [groups, beams] (undefined: no beam is).  A finished beam goes on with the token eos at its score;
// eos < 0: no token ends a sequence.
BeamStep beam_select(const Tensor& logits, const Tensor& scores, const Tensor& finished, int eos = -1);

}  // namespace Inferno
