"""CPU: the tuning operators (losses from logits, embedding, gradient clipping) refuse wrong arguments before any device work, in Python and at the
C entries."""
import pytest
import torch


def _logits(B=2, T=3, V=5, dtype=torch.float32):
    return torch.zeros(B, T, V, dtype=dtype), torch.zeros(B, T, dtype=torch.int64)


def test_cpu_tensors_are_refused():
    from bmt_amd import ops
    from bmt_amd.loss.policy import PolicyLoss, PreferenceLoss
    from bmt_amd.optim import GradClipper
    x, ids = _logits()
    row = torch.zeros(2, 3)
    for call in (lambda: ops.token_logp(x, ids), lambda: PolicyLoss(pad_idx=1)(x, ids, row, row), lambda: PreferenceLoss()(x, ids, torch.zeros(2)),
                 lambda: ops.embedding(ids, torch.zeros(4, 5)), lambda: GradClipper([torch.zeros(3)], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("change", ["rank", "ids_shape", "ids_type", "dtype", "mask_shape", "mask_type", "empty_vocabulary"])
def test_rows_of_the_wrong_kind_are_refused(change):
    from bmt_amd import ops
    x, ids = _logits()
    mask = torch.ones(2, 3, dtype=torch.bool)
    if change == "rank":
        x = x[0]
    elif change == "ids_shape":
        ids = ids[:, :-1]
    elif change == "ids_type":
        ids = ids.int()
    elif change == "dtype":
        x = x.double()
    elif change == "mask_shape":
        mask = mask[:1]
    elif change == "mask_type":
        mask = mask.float()
    else:
        x = x[:, :, :0]
    row = torch.zeros(2, 3)
    for call in (lambda: ops.token_logp(x, ids, mask), lambda: ops.policy_loss(x, ids, row, row, mask=mask), lambda: ops.preference_loss(x, ids, torch.zeros(2), mask)):
        with pytest.raises(ValueError):
            call()


def test_c_entries_refuse_before_any_launch():
    from bmt_amd import _lib
    lib = _lib.load()
    some = 4096      # (an address that is never followed: every call below is refused on its sizes, types, alignments or null pointers)
    rows = lambda x=some, dtype=0, sb=15, st=5, B=2, T=3, V=5, ids=some: (x, dtype, sb, st, B, T, V, ids, 3, 1, None, 0, 0, -1)      # noqa: E731
    for bad in (dict(x=None), dict(dtype=3), dict(V=0), dict(B=-1), dict(ids=None), dict(x=some + 2), dict(sb=-1), dict(B=1 << 20, T=1 << 20)):
        assert lib.bmt_logp_rows(*rows(**bad), some, some, None) == -1 and b"bmt_logp_rows" in lib.bmt_last_error(), bad
    assert lib.bmt_logp_rows(*rows(B=0), None, None, None) == 0
    assert lib.bmt_logit_grad(*rows(), None, some, 1, 1, None, 0, some, 15, 5, None) == -1
    assert lib.bmt_logit_grad(*rows(), some, some, 1, 1, None, 0, some + 1, 15, 5, None) == -1

    def policy(ws_bytes=None, ws=some, reduction=1, lo=0.2, adv=some, d=None, **kw):
        n = lib.bmt_policy_ws_bytes(2, 3) if ws_bytes is None else ws_bytes
        return lib.bmt_policy_loss(*rows(**kw), some, 3, 1, None, 0, 0, adv, 1, 0, lo, 0.2, 0.0, reduction, some, some, some, ws, n, d, 15, 5, None)
    for bad in (dict(ws_bytes=lib.bmt_policy_ws_bytes(2, 3) - 1), dict(ws=some + 8), dict(reduction=3), dict(lo=-0.1), dict(adv=None), dict(B=0), dict(d=some + 2)):
        assert policy(**bad) == -1 and b"bmt_policy_loss" in lib.bmt_last_error(), bad

    def preference(ws_bytes=None, smoothing=0.0, ref=some, **kw):
        n = lib.bmt_preference_ws_bytes(2, 3) if ws_bytes is None else ws_bytes
        return lib.bmt_preference_loss(*rows(**kw), ref, 1, 0.1, smoothing, 0, some, some, some, n, None)
    for bad in (dict(ws_bytes=8), dict(smoothing=1.5), dict(smoothing=float("nan")), dict(ref=None), dict(B=3), dict(T=0)):
        assert preference(**bad) == -1 and b"bmt_preference_loss" in lib.bmt_last_error(), bad

    assert lib.bmt_embedding(None, None, 4, None, 0, 4, 4, 0, 1.0, None) == 0
    for bad in ((some, some, 3, some, 2, 4, 4, 0), (some, some, 4, some, 2, 0, 4, 0), (some, some, 4, some, 2, 4, 4, 5), (None, some, 4, some, 2, 4, 4, 0)):
        assert lib.bmt_embedding(*bad, 1.0, None) == -1 and b"bmt_embedding" in lib.bmt_last_error(), bad
    n = lib.bmt_embedding_bwd_ws_bytes(100, 6, 9)
    assert n >= (9 + 1 + 2 * 100) * 4 and lib.bmt_embedding_bwd_ws_bytes(1 << 31, 6, 9) == 0

    def bwd(dtype=0, dW=some, into=None, ws=some, ws_bytes=n, N=100, ids=some):
        return lib.bmt_embedding_bwd(ids, some, 6, N, 6, 9, dtype, 1.0, -1, dW, into, 6, ws, ws_bytes, None)
    for bad in (dict(dtype=7), dict(dW=None), dict(into=some), dict(dtype=1, dW=None, into=some), dict(ws=some + 8), dict(ws_bytes=n - 1), dict(N=-1), dict(ids=None)):
        assert bwd(**bad) == -1 and b"bmt_embedding_bwd" in lib.bmt_last_error(), bad

    n = lib.bmt_clip_ws_bytes()
    assert lib.bmt_clip_tile_bytes() == 24
    for bad in ((None, 1, some, some, n), (some, 1, None, some, n), (some, 1, some, None, n), (some, 1, some, some, n - 1), (some + 4, 1, some, some, n), (some, -1, some, some, n)):
        assert lib.bmt_clip_grads(bad[0], bad[1], 0, 1.0, 1e-6, None, 1, 0, *bad[2:], None) == -1 and b"bmt_clip_grads" in lib.bmt_last_error(), bad


def test_gradient_layouts_are_dense_or_refused():
    from bmt_amd.optim import _dense
    t = torch.zeros(4, 6)
    assert _dense(t) and _dense(t.t()) and _dense(t[1:3]) and _dense(torch.zeros(())) and _dense(torch.zeros(2, 3, 4).permute(2, 0, 1)) and _dense(t[:, :1][:1])
    assert not _dense(t[:, :3]) and not _dense(t[::2]) and not _dense(torch.zeros(1, 6).expand(4, 6))


def test_calls_that_no_grid_holds_are_refused():
    """a launch has fewer than 2^32 threads: 64 for a short row, 256 for four tokens of a lookup or of a table"""
    from bmt_amd import _lib
    lib = _lib.load()
    some = 4096
    assert lib.bmt_logp_rows(some, 0, 5 << 13, 5, 1 << 14, 1 << 13, 5, some, 1 << 13, 1, None, 0, 0, -1, some, some, None) == -1
    assert b"more than a grid holds" in lib.bmt_last_error()
    assert lib.bmt_embedding(some, some, 64, some, 1 << 31, 64, 1000, 0, 1.0, None) == -1 and b"more than a grid holds" in lib.bmt_last_error()
    V = 1 << 30
    n = lib.bmt_embedding_bwd_ws_bytes(100, 6, V)
    assert lib.bmt_embedding_bwd(some, some, 6, 100, 6, V, 0, 1.0, -1, some, None, 6, some, n, None) == -1 and b"more than a grid holds" in lib.bmt_last_error()
