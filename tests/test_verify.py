"""``verify_drafts`` without a GPU: what is refused before a launch."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from llm_serving_layer_amd import _native, sampling

from ._verify import verify64


def test_the_oracle_on_rows_by_hand():
    """p = (1/4, 1/2, 1/4): a draft of token 1 under q = 1 falls at 0.5, the rest
    halves between 0 and 2; under q = (0, 1, 0) likewise."""
    logits = torch.tensor([[0.0, 0.6931471805599453, 0.0]], dtype=torch.float64).expand(2, 3)
    tokens = torch.tensor([0, 1])
    for probs in (None, torch.tensor([[0.0, 1.0, 0.0]])):
        for u, last, want in [(0.49, 0.3, ([1, 1], 1)), (0.51, 0.49, ([0, -1], 0)),
                              (0.51, 0.51, ([2, -1], 0)), (0.49, 0.2, ([1, 0], 1))]:
            ids, n, _ = verify64(logits, tokens, [2], torch.tensor([u, last]), probs)
            assert (ids[0].tolist(), int(n[0])) == want


@pytest.mark.parametrize("logits,match", [
    (torch.zeros(3), "must be \\(n_tokens, vocab\\)"), (torch.zeros(3, 4), "on the GPU")])
def test_bad_logits_are_refused(logits, match):
    with pytest.raises(ValueError, match=match):
        sampling.verify_drafts(logits, None, None, None)


BASE = dict(logits=256, n_rows=3, vocab=10, stride=10, dtype=0, tokens=256, cu=256, owner=256,
            n_seqs=2, numbers=256, probs=None, pstride=0, pdtype=0, temps=None, temp=1.0, ids=256,
            width=2, accepted=256, ws=256, ws_bytes=1 << 20)


@pytest.mark.parametrize("change,match", [
    ({"dtype": 7}, "dtype"), ({"vocab": 0}, "vocab"), ({"vocab": 2**31}, "vocab"),
    ({"n_seqs": 0}, "sequences"), ({"n_seqs": 4}, "sequences"), ({"stride": 9}, "row_stride"),
    ({"probs": 256, "pdtype": 9}, "probs_dtype"), ({"width": 0}, "width"), ({"width": 4}, "width"),
    ({"probs": 256, "pstride": 5, "n_rows": 4}, "probs_stride"), ({"numbers": None}, "null"),
    ({"ws": None}, "null"), ({"ws_bytes": 16}, "workspace"), ({"ws": 264}, "workspace")])
def test_the_entry_refuses(change, match):
    a = {**BASE, **change}
    rc = _native.load().pkv_verify_drafts(*a.values(), None)
    with pytest.raises(ValueError, match=match):
        _native.check(rc, "verify")


@pytest.mark.parametrize("rows,seqs,vocab", [(1, 1, 1), (5, 1, 128256), (249, 64, 128256),
                                             (100000, 50000, 12)])
def test_the_workspace_grows_with_the_batch(rows, seqs, vocab):
    size = _native.load().pkv_verify_workspace_bytes
    one = size(rows, seqs, vocab, 0)
    assert one >= 16 * rows + 24 * seqs
    assert size(rows, seqs, vocab, 9) == size(0, 1, vocab, 0) == size(rows, seqs, 0, 0) == 0
    assert C.c_int64(one).value == one
