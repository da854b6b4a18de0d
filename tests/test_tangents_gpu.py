"""Forward-mode derivatives of the flash attention, the similarity and the polar transform: there are none, and a transform that asks for
them is told so, where torch's ops would give tangents of 0."""
import pytest
import torch

from pope_amd import apply_pope_to_qk
from pope_amd.attention import flash_attn_with_pope
from pope_amd.hip_pope import hip_compute_qk_similarity

pytestmark = pytest.mark.gpu

CALLS = {"flash": lambda q, k, v, f, b: flash_attn_with_pope(q, k, v, (f, b)), "similarity": lambda q, k, v, f, b: hip_compute_qk_similarity(q, k, f, b),
         "polar": lambda q, k, v, f, b: torch.cat([t.flatten() for t in apply_pope_to_qk((f, b), q, k)])}


@pytest.mark.parametrize("dims", [(64, 32), (40, 20)])
@pytest.mark.parametrize("call", CALLS)
def test_tangents_are_refused(cuda, call, dims):
    D, R = dims
    args = [torch.randn(2, 4, 70, D, device=cuda) for _ in range(3)] + [torch.rand(70, R, device=cuda), -torch.rand(4, R, device=cuda)]
    for i in range(5):
        if call != "flash" and i == 2:
            continue
        f = lambda t: CALLS[call](*args[:i], t, *args[i + 1:])
        with pytest.raises((RuntimeError, NotImplementedError), match="forward-mode|forward mode"):
            torch.func.jvp(f, (args[i],), (torch.ones_like(args[i]),))
    out = CALLS[call](*args)
    assert torch.equal(torch.func.vmap(lambda b: CALLS[call](*args[:4], b))(args[4][None])[0], out)   # other transforms are as they were
