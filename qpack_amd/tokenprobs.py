"""logprobs: log probabilities of given tokens, entropy, ranks and alternatives over the C ABI (qph_logprobs), for torch tensors on the GPU."""
from collections import namedtuple

# logp: of the given tokens; entropy in nats; rank: the number of tokens ahead (0: the most probable); top_index, top_logp [rows][top]: the first ones in that order
LogProbs = namedtuple("LogProbs", "logp entropy rank top_index top_logp")


def logprobs(logits, tokens=None, top=0):
    """LogProbs of the rows of logits [rows, vocab] (float32, float16 or bfloat16, each row contiguous) and of tokens (int32 [rows]): tensors, in one pass over
    the logits, on the current stream of their device and not waited for; can be captured into a graph.

    A token outside the vocabulary has logp NaN and rank -1; without tokens logp and rank are None.  top <= 64.  Of equal logits the lower index
    comes first.  Logits of -inf have probability 0; a row with a NaN or +inf, or of -inf alone, has NaN results.  Nothing here carries gradients: logits that
    require one are refused while gradients are recorded, and those with a forward-mode tangent.  The results lie side by side in one allocation."""
    from .kvcache import _binding
    return LogProbs(*_binding().logprobs(logits, tokens, top))
