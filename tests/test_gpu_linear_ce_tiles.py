"""The projection's cross entropy at sizes that take each of its tiles, tiles shared between
workgroups, and several pieces of the vocabulary, against the oracle."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).parent))
from test_gpu_linear_ce import _check, _make  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_tiles_of_256(dtype):
    """All three products on 256 x 256 tiles, none of whose sizes is a multiple of 256."""
    _check(*_make(4003, 2000, 20001, dtype, 0.02))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens,hidden,vocab", [
    (17, 1032, 700), (1, 4104, 66), (100, 1000, 3000), (129, 520, 40000), (1500, 264, 2500),
    (2500, 96, 30000), (70, 72, 70000)])
def test_other_tiles(dtype, tokens, hidden, vocab):
    _check(*_make(tokens, hidden, vocab, dtype, 0.05), smoothing=0.1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ignored", [0.5, 0.9, 0.97, 0.9995])
def test_few_of_many_tokens_count(dtype, ignored):
    """Tiles of dx shared by as many workgroups as the tokens that count leave room for."""
    _check(*_make(3001, 520, 9001, dtype, ignored))


@pytest.mark.parametrize("ignored", [0.0, 0.99])
def test_pieces_shared_between_workgroups(ignored):
    """Several pieces of the vocabulary: sums of dx onto those of the pieces before, and a last
    piece with fewer columns than workgroups share."""
    _check(*_make(20001, 64, 16100, BF16, ignored))
    _check(*_make(20001, 32, 8230, F32, ignored))
