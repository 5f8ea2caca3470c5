"""The operands of tests/test_gpu_act8_exact.py notice what is left out of a weight gradient: on the
CPU, results with something missing are rejected."""
import pytest
import torch

import _act8exact as ex

F32, BF16 = torch.float32, torch.bfloat16


def _rejected(got, want):
    with pytest.raises(AssertionError):
        ex.same(got, want, "")


@pytest.mark.parametrize("T,N,K,dtype", [(65, 127, 129, BF16), (5000, 40, 64, BF16), (5000, 95, 96, F32),
                                         (100000, 18, 20, BF16)])
def test_whole_numbers_notice_missing_tokens(T, N, K, dtype):
    gy, q, scale, dw, db = ex.whole(T, N, K, dtype, 1, "cpu")
    for out in (F32, BF16):
        ex.same(dw.to(F32).to(out), dw, "dw")
        ex.same(db.to(F32).to(out), db, "db")
        _rejected(torch.zeros(N, K, dtype=out), dw)
    for cut in (slice(64, None), slice(0, T - 1), slice(0, T - T % 64 if T % 64 else T - 64)):
        w, b = ex.product(gy[cut], q[cut], scale[cut], K)
        _rejected(w.to(F32), dw)
        _rejected(b.to(F32), db)
    # in another order, in float32: the same
    order = torch.randperm(T, generator=torch.Generator().manual_seed(2))
    ex.same(gy[order].float().t() @ ex._values(q, scale, K)[order].float(), dw, "dw")


@pytest.mark.parametrize("T,N,K", [(65, 130, 130), (5000, 95, 96)])
def test_parts_notice_missing_parts_and_tokens(T, N, K):
    gy, q, scale, dw, db = ex.parts(T, N, K, 1, "cpu")
    assert int((gy != 0).sum()) == N

    def cut(v):
        return (v.view(torch.int32) & -65536).view(F32)          # the upper half: a bf16 by truncation

    hi = cut(gy)
    mid = cut(gy - hi)
    lo = gy - hi - mid
    assert torch.equal(cut(lo), lo)                              # three parts hold a float32
    ex.same(sum(ex.product(p, q, scale, K)[0] for p in (hi, mid, lo)).float(), dw, "dw")
    for some in (hi, hi + mid, hi + lo, mid + lo):
        w, b = ex.product(some, q, scale, K)
        _rejected(w.float(), dw)
        _rejected(b.float(), db)
    w, b = ex.product(gy[64:], q[64:], scale[64:], K)
    _rejected(w.float(), dw)
    _rejected(b.float(), db)
