"""Calls that reach every kernel of the norms' gradients and of the projection's cross entropy at
sizes whose last vectors, tiles, stages and pieces are not full.  run() returns the outputs; as a
program it saves them, and the debug library's failed bounds checks, to the file it is given."""
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
NORMS = [(3, 5), (129, 40), (513, 100), (4097, 33), (258, 768), (5003, 1001), (300, 4096),
         (33, 9000), (20, 20480), (19, 20481), (9, 30000), (6, 40000)]
# tokens, hidden, classes, share of tokens ignored
LOSSES = [(1, 1, 1, 0.0), (3, 33, 5, 0.0), (31, 100, 1000, 0.3), (64, 72, 130, 0.0),
          (65, 128, 300, 0.3), (300, 768, 5003, 0.4), (1000, 512, 9000, 0.0), (70, 30, 30, 1.0),
          (4003, 2000, 20001, 0.02), (20001, 64, 16100, 0.99)]


def _bits(t):
    whole = t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)
    return whole.long().sum().cpu()


def run() -> dict:
    out = {}
    for dtype in (torch.float32, torch.bfloat16):
        g = torch.Generator(DEV).manual_seed(1)
        for rows, cols in NORMS:
            x, dy = (torch.randn(rows, cols, generator=g, device=DEV).to(dtype) for _ in range(2))
            w = (torch.rand(cols, generator=g, device=DEV) + 0.5).to(dtype)
            got = [*layer_norm_bwd(dy, x, w, w), *rms_norm_bwd(dy, x, (cols,), w)]
            for i, t in enumerate(got):
                out[f"norm {dtype} {rows} {cols} {i}"] = _bits(t)
        for tokens, hidden, vocab, ignored in LOSSES:
            if dtype == torch.float32 and tokens > 2000:
                continue
            x = torch.randn(tokens, hidden, generator=g, device=DEV).to(dtype)
            w = torch.randn(vocab, hidden, generator=g, device=DEV).to(dtype)
            lab = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
            lab[torch.rand(tokens, generator=g, device=DEV) < ignored] = -100
            dloss = torch.rand(tokens, generator=g, device=DEV)
            loss, lse, z = linear_cross_entropy_fwd(x, w, lab, smoothing=0.1)
            got = [loss, lse, z, *linear_cross_entropy_bwd(dloss, x, w, lse, lab, smoothing=0.1)]
            for i, t in enumerate(got):
                out[f"loss {dtype} {tokens} {hidden} {vocab} {i}"] = _bits(t)
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
