"""Calls of the norms' gradients whose workgroups go over several rows (the next one's loads ahead),
and of the projection's gradients in fp16 with losses of very different weights.  run() returns the
outputs; as a program it saves them, and the debug library's failed bounds checks, to the file it is
given."""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from dslperfgap_amd import _lib  # noqa: E402
from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd  # noqa: E402
from dslperfgap_amd.viperbench.linear_cross_entropy.hip_impl import (  # noqa: E402
    linear_cross_entropy_bwd, linear_cross_entropy_fwd)
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd  # noqa: E402

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NORMS = [(BF16, 513, 20480), (BF16, 520, 24576), (F16, 515, 32768), (BF16, 513, 20481),
         (F16, 514, 30001), (F32, 515, 12288), (F32, 513, 16384), (F32, 514, 9001), (F32, 3, 70001)]
# tokens, hidden, classes, share of tokens ignored
LOSSES = [(1, 1, 1, 0.0), (3, 33, 5, 0.0), (31, 100, 1003, 0.3), (300, 768, 5003, 0.4),
          (300, 64, 301, 0.0), (70, 30, 30, 1.0), (4003, 520, 12001, 0.02), (20001, 64, 16100, 0.5)]


def _bits(t):
    whole = t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)
    flat = whole.reshape(-1).long()
    # values in each other's places count
    return (flat * (1 + torch.arange(flat.numel(), device=DEV) % 8191)).sum().cpu()


def run() -> dict:
    out = {}
    g = torch.Generator(DEV).manual_seed(1)
    for dtype, rows, cols in NORMS:
        x, dy = (torch.randn(rows, cols, generator=g, device=DEV).to(dtype) for _ in range(2))
        w = (torch.rand(cols, generator=g, device=DEV) + 0.5).to(dtype)
        if dtype != F16:  # rows that are gone over once more
            x[::3] *= 1e16
            dy[::3] *= 1e23
        got = [*layer_norm_bwd(dy, x, w, w), *rms_norm_bwd(dy, x, (cols,), w)]
        for i, t in enumerate(got):
            out[f"norm {dtype} {rows} {cols} {i}"] = _bits(t)
    for tokens, hidden, vocab, ignored in LOSSES:
        x = torch.randn(tokens, hidden, generator=g, device=DEV).to(F16)
        w = torch.randn(vocab, hidden, generator=g, device=DEV).to(F16)
        lab = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
        lab[torch.rand(tokens, generator=g, device=DEV) < ignored] = -100
        dloss = torch.exp2(-24 * torch.rand(tokens, generator=g, device=DEV))
        lse = linear_cross_entropy_fwd(x, w, lab)[1]
        got = linear_cross_entropy_bwd(dloss, x, w, lse, lab)
        for i, t in enumerate((lse, *got)):
            out[f"loss {tokens} {hidden} {vocab} {i}"] = _bits(t)
    torch.cuda.synchronize()
    return out


if __name__ == "__main__":
    # child process: VBHIP_LIB names the debug library
    _lib.lib()
    _lib.debug_bounds(clear=True)
    outs = run()
    failed, where = _lib.debug_bounds(clear=True)
    torch.save({"outs": outs, "failed": failed, "where": where}, sys.argv[1])
    print(f"[bounds] {len(outs)} outputs, {failed} failed checks", flush=True)
