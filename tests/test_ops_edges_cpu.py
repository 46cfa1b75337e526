"""Calls of the operators around attention at the edge of what they document, as far
as a machine without a GPU shows it."""
import pytest
import torch
import torch.autograd.forward_ad as ad

import flash_attention_v100 as fa


def test_forward_mode_derivatives_are_refused():
    # before anything else is looked at: without the refusal the result has no tangent
    q, k, v = (torch.zeros(1, 4, 2, 8) for _ in range(3))
    table = torch.zeros(4, 8)
    for f, args in ((fa.flash_attention_v100_scored, (q, k, v)), (fa.rotary_embedding_v100, (q, k, table)),
                    (lambda q, k, v: fa.flash_attention_v100_shared_prefix(q, k[0], v[0], k, v), (q, k, v))):
        for i in range(len(args)):
            with ad.dual_level(), torch.no_grad():
                dual = [ad.make_dual(t, torch.ones_like(t)) if n == i else t for n, t in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*dual)
                with ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="no CPU path"):
                    f(*dual)
            with pytest.raises(ValueError, match="no CPU path"):
                f(*args)
