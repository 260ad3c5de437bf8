"""RMS norm of query and key heads with the position rotation in the same pass, forward and backward."""
import torch  # noqa: F401  (in front of the extension, which links against it)

import vllm_flash_attn_2_cuda as flash_attn_cuda


def qk_norm_rotary_func(q, k, q_weight, k_weight, rotary_cos, rotary_sin, positions=None, eps=1e-6, rotary_interleaved=True):
    """RMS norm of every head of q (batch_size, seqlen, nheads, headdim) and k (batch_size, seqlen, nheads_k, headdim), times
    q_weight / k_weight (headdim,), then the rotation of the first rotary_dim columns by the token's position:

        y = R(position) (x / sqrt(mean(x^2) + eps) * weight)

    rotary_cos / rotary_sin (seqlen_ro, rotary_dim / 2) turn the pairs (2i, 2i + 1) if rotary_interleaved, else
    (i, i + rotary_dim / 2), like those of flash_attn_with_kvcache; rotary_dim is a multiple of 16.  Weights and tables are
    fp32 or of q's type; sums and products are fp32 and the result is rounded once.  positions (batch_size, seqlen) int32
    defaults to 0 .. seqlen - 1; a negative position marks padding (output and gradients are zero there), one past the
    tables gives NaN.  A ragged batch is q (total, nheads, headdim), k (total, nheads_k, headdim) with positions (total,).

    Returns (q_out, k_out).  Differentiable in q, k and the weights (not in the tables; an input with a forward-mode
    tangent is refused); gradients are bitwise reproducible.  Can be captured into a graph with its backward, unless a graph recorded on the default stream still
    holds one of the inputs or what it is a view of (refused: the backward pass would end the process).  headdim is a
    multiple of 8, at most 256.  No counterpart in the reference, whose cache call rotates q and k
    (csrc/flash_attn/src/rotary.h:19-148) but does not norm them."""
    ragged = q.dim() == 3
    if ragged:
        if positions is None:
            raise ValueError("positions are required with ragged q and k")
        q, k, positions = q[None], k[None], positions[None]
    if positions is not None and positions.stride(-1) != 1:
        positions = positions.contiguous()
    if rotary_cos.requires_grad or rotary_sin.requires_grad:
        raise ValueError("rotary_cos and rotary_sin have no gradient: detach them")
    out = flash_attn_cuda.qk_norm_rotary(q, k, q_weight, k_weight, rotary_cos, rotary_sin, positions, eps, rotary_interleaved)
    return tuple(x[0] for x in out) if ragged else tuple(out)
