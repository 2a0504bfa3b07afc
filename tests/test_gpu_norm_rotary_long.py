"""norm_rotary_embed on an MI355X with more tokens than the backward's workgroups take in one step, against the float64
oracle, element by element within its bounds."""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

from oracle import norm_rotary_ref as NR
from rfdetr_jax_amd import norm_rotary_embed

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _np(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tokens", [16384, 16385, 16400, 18433, 33000])
@pytest.mark.parametrize("dim", [16, 10])  # rows on 16-byte boundaries, and others
def test_many_tokens(dim, tokens, dtype):
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    sys.stderr.write(f"[gpu] norms with rotary positions, {tokens} tokens of {dim} channels {dtype}\n")
    g, sections = torch.Generator().manual_seed(tokens), (dim // 2,)
    made = [torch.randn(s, generator=g).to(dtype).cuda() for s in ((tokens, 2, dim), (tokens, 1, dim), (dim,), (dim,), (tokens, 2, dim), (tokens, 1, dim))]
    leaves, cotangents = [x.requires_grad_(True) for x in made[:4]], made[4:]
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")[:, None]
    outs = norm_rotary_embed(*leaves, pos, sections)
    grads = torch.autograd.grad(outs, leaves, cotangents)
    u, p = HALF_STEP[dtype], pos.cpu().numpy()
    options = {"shared": False, "interleaved": False, "base": 10000.0}
    for i in range(2):
        args = (_np(leaves[i]), _np(leaves[2 + i]), p, sections, 1e-6)
        pairs = [(outs[i], NR.forward(*args, **options), NR.forward_bound(*args, u, **options))]
        args = (_np(leaves[i]), _np(leaves[2 + i]), _np(cotangents[i]), p, sections, 1e-6)
        pairs += list(zip((grads[i], grads[2 + i]), NR.backward(*args, **options), NR.backward_bounds(*args, u, u, **options)))
        for got, want, bound in pairs:
            assert got.shape == want.shape and got.dtype == dtype
            assert (np.abs(_np(got) - want) <= bound).all()
