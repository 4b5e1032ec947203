"""The rotation over more waves than one launch may have: it takes two launches, which meet
in the middle of the tokens."""
import pytest
import torch

from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
from dslperfgap_amd.viperbench.rope.hip_impl import rope_bwd, rope_fwd
from oracle import rope as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
# a token's queries and keys take a wave each; a launch has fewer than 2^32 lanes, 2^26 waves
TOKENS = 36_000_001


@pytest.mark.parametrize("dim,pairing", [(2, "half"), (2, "adjacent"), (3, "half")])
def test_more_tokens_than_one_launch_takes(dim, pairing):
    """The same bits as two calls that each fit one launch."""
    print(f"[gpu] {TOKENS} tokens, heads of {dim}, {pairing}", flush=True)
    g = torch.Generator(DEV).manual_seed(dim)
    q, k, gq, gk = (torch.randn(TOKENS, 1, dim, generator=g, device=DEV) for _ in range(4))
    pos = torch.randint(0, 5000, (TOKENS,), generator=g, device=DEV, dtype=torch.int32)
    freq, w = ref.inv_freq(1).to(DEV), torch.linspace(0.5, 1.5, dim, device=DEV)
    how = {"pairing": pairing}
    halves = slice(0, TOKENS // 2), slice(TOKENS // 2, TOKENS)

    def same(fn, *x, args=(), n=2):
        whole = fn(*x, *args, pos, freq, **how)
        for h in halves:
            part = fn(*[t[h] for t in x], *args, pos[h], freq, **how)
            assert all(torch.equal(a[h], b) for a, b in zip(whole[:n], part[:n])), h
        return whole

    same(rope_fwd, q, k)
    same(rope_bwd, gq, gk)
    same(qk_norm_rope_fwd, q, k, args=(w, w))
    same(qk_norm_rope_bwd, gq, gk, q, k, args=(w, w))
