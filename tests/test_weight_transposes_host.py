"""The batched transposes of the token Linears' weights (linear._WT) without a GPU: which requests a
launch takes.  The launch is recorded, not made."""
import gc

import pytest
import torch

from visionseg import linear, ops


@pytest.fixture
def wt(monkeypatch):
    """-> (the batch, the launches so far as lists of written buffers, a cell with the current place)"""
    launches, place = [], ["stream 1"]

    def write(pairs):
        for src, dst in pairs:
            dst.copy_(src.t())
        launches.append([dst for _, dst in pairs])

    monkeypatch.setattr(ops, "transpose_batched", write)
    monkeypatch.setattr(linear, "_place", lambda w: place[0], raising=False)
    return linear._WeightTransposes(), launches, place


def _w(k):
    return torch.randn(3, 5, generator=torch.Generator().manual_seed(k))


def test_one_launch_writes_the_requests_of_a_place(wt):
    batch, launches, _ = wt
    ws = [_w(k) for k in range(4)]
    hs = [batch.request(w) for w in ws]
    assert [torch.equal(batch.get(h), w.t()) for h, w in zip(hs[::-1], ws[::-1])] == [True] * 4
    assert [len(l) for l in launches] == [4] and not batch.pending


def test_another_place_is_left_alone(wt):
    """Another stream, or eager work while a capture records: what the launch writes is not ordered
    before, or not run before, the other's use."""
    batch, launches, place = wt
    a, b = _w(1), _w(2)
    ha = batch.request(a)
    place[0] = "stream 2"
    hb = batch.request(b)
    assert torch.equal(batch.get(hb), b.t())
    assert [len(l) for l in launches] == [1]                  # b alone
    place[0] = "stream 1"
    assert torch.equal(batch.get(ha), a.t()) and [len(l) for l in launches] == [1, 1]
    # a backward elsewhere than its forward: a copy of its own, before and after the batch is written
    hc, hd = batch.request(a), batch.request(b)
    place[0] = "capture"
    assert torch.equal(batch.get(hc), a.t()) and len(launches) == 2
    place[0] = "stream 1"
    assert torch.equal(batch.get(hd), b.t()) and len(launches) == 3
    place[0] = "capture"
    assert torch.equal(batch.get(hd), b.t()) and batch.get(hd).data_ptr() != launches[2][-1].data_ptr()


def test_a_forward_without_a_backward_leaves_nothing(wt):
    """A captured launch that wrote into a dead request's buffer would do so at every replay."""
    batch, launches, _ = wt
    dropped = batch.request(_w(1))
    kept = batch.request(_w(2))
    buffer = dropped if isinstance(dropped, list) else dropped.out
    del dropped, buffer
    gc.collect()
    assert len(batch.pending) == 1
    batch.get(kept)
    assert [len(l) for l in launches] == [1]
    for k in range(2000):
        batch.request(_w(3))
    assert not batch.pending


def test_two_threads(wt):
    """Forwards of one thread while another runs backwards: every get() is the transpose."""
    import sys
    import threading
    batch, _, _ = wt
    ws = [_w(k) for k in range(8)]
    queue, errors, turns = [], [], 3000

    def forwards():
        for k in range(turns):
            queue.append((batch.request(ws[k % 8]), ws[k % 8]))

    def backwards():
        done = 0
        while done < turns and not errors:
            if queue:
                h, w = queue.pop(0)
                if not torch.equal(batch.get(h), w.t()):
                    errors.append(done)
                done += 1

    def guarded(f):
        try:
            f()
        except Exception as e:
            errors.append(e)

    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=guarded, args=(f,)) for f in (forwards, backwards)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
    finally:
        sys.setswitchinterval(before)
    assert not errors, errors[:3]
