"""Token embedding with a scale on the HIP engine (the reference's nn.Embedding, models/lm.py:125).

The gradient sorts the tokens on the GPU and adds the rows that belong to one token in their order: nothing is
read back on the host, so a training step can be captured in a HIP graph, and the sums are the same every time.
"""

from . import _abi


def embedding(tokens, weight, scale=1.0):
    """scale * weight[tokens], (..., C) in weight's type.

    tokens (...): integers; a token outside [0, vocabulary), as -1 for padding, gives a row of zeros and no
    gradient.  weight (vocabulary, C) float32, bfloat16 or float16.  Differentiable (reverse mode) in weight, any number
    of times; the gradient is dense, summed in float32, of fewer than 2^27 tokens."""
    return _abi.host().embedding(tokens, weight, float(scale))
