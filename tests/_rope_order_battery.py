"""Calls of the query / key operators whose outputs are kept as two checksums that see a
value in another's place: the bits times odd factors that differ from place to place, summed
in 64 bits.  Some vectors hold the type's lowest value, so that the backward goes over its
shares twice.  run() returns the checksums (of fp32 and bf16); as a program it saves them, and the debug
library's failed bounds checks, to the file it is given."""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from dslperfgap_amd import _lib  # noqa: E402
from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import (  # noqa: E402
    qk_norm_rope_bwd, qk_norm_rope_fwd)
from dslperfgap_amd.viperbench.rope.hip_impl import rope_bwd, rope_fwd  # noqa: E402

DEV = "cuda:0"
SIZES = [(64, 32), (64, 20), (72, 36), (80, 40), (96, 48), (100, 50), (50, 25), (33, 16),
         (130, 65), (192, 96), (256, 128), (1023, 511), (1024, 512)]
# tokens, query heads, key heads: single passes; shares of several, several tokens a wave
COUNTS = [(1, 1, 1), (37, 5, 2), (8193, 9, 3)]


def checksums(t) -> list:
    bits = t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)
    bits = bits.reshape(-1).long()
    at = torch.arange(bits.numel(), device=bits.device)
    # odd multiples of 64-bit constants: another factor in every place
    return [int((bits * ((2 * at + 1) * c)).sum())
            for c in (0x1E3779B97F4A7C15, 0x3C6EF372FE94F82B)]


def run() -> dict:
    out = {}
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for dim, n in SIZES:
            for tokens, hq, hk in COUNTS:
                if tokens > 1000 and dim > 256:
                    continue
                g = torch.Generator(DEV).manual_seed(dim + tokens)

                def heads(h):
                    return torch.randn(tokens, h, dim, generator=g, device=DEV).to(dtype)

                q, k, gq, gk = heads(hq), heads(hk), heads(hq), heads(hk)
                low = [torch.rand(t.shape[:2], generator=g, device=DEV) < 0.02 for t in (q, k)]
                qn, kn = q.clone(), k.clone()
                qn[low[0]] = kn[low[1]] = torch.finfo(dtype).min
                w = torch.rand(dim, generator=g, device=DEV) + 0.5
                pos = torch.arange(tokens, device=DEV)
                freq = 10000.0 ** -(torch.arange(n, device=DEV) / n)
                for pairing in ("half", "adjacent"):
                    key = f"{dtype} {dim} {n} {tokens} {pairing} "
                    got = [*rope_fwd(q, k, pos, freq, pairing=pairing),
                           *rope_bwd(gq, gk, pos, freq, pairing=pairing),
                           *qk_norm_rope_fwd(qn, kn, w, w, pos, freq, pairing=pairing),
                           *qk_norm_rope_bwd(gq, gk, qn, kn, w, w, pos, freq, pairing=pairing)]
                    if dtype == torch.float16:
                        # only for the bounds checks: whether a fused multiply-add and the
                        # rounding to 16 bits are one instruction (v_fma_mix), which rounds
                        # once, or two is the compiler's choice in each of the libraries
                        continue
                    for i, t in enumerate(got):
                        out[key + str(i)] = checksums(t)
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
