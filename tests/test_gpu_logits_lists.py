"""Bias lists that name tokens many times: the values against numpy's own additions in list order, bit for bit, and their cost against lists that name each token once."""
import numpy as np
import pytest
import torch

import lithos_metal_b200 as lm

pytestmark = pytest.mark.gpu


def repeated(rng, kind, vocab, n):
    ids = rng.permutation(vocab)[:n].astype(np.int32)
    values = rng.normal(0, 4, n).astype(np.float32)
    if kind == "padded":                                                      # with a valid id and nothing to add
        ids[n // 5:], values[n // 5:] = 3, 0.0
    elif kind == "equal":
        ids[:] = vocab - 1
    elif kind == "twice":
        ids[n // 2:2 * (n // 2)] = ids[: n // 2][rng.permutation(n // 2)]
    elif kind == "runs":                                                      # one token many times in some warps, few of it in others
        ids = np.sort(rng.integers(0, max(2, n // 20), n)).astype(np.int32)
        ids[::50] = 0
    return ids, values


def added(z, ids, values):
    """float32 additions in list order."""
    z = z.copy()
    for i, v in zip(ids.tolist(), values):
        z[i] = np.float32(z[i] + v)
    return z


@pytest.mark.parametrize("place", ["new", "same"])
@pytest.mark.parametrize("history", [False, True])
@pytest.mark.parametrize("n", [2, 33, 300, 1200, 8191])
@pytest.mark.parametrize("kind", ["padded", "equal", "twice", "runs"])
def test_values_are_added_once_in_list_order(kind, n, history, place):
    rng = np.random.default_rng(n)
    vocab = 20_011
    z = (rng.standard_normal((3, vocab)) * 3).astype(np.float32)
    lists = [repeated(rng, kind, vocab, n) for _ in range(3)]
    want = z.copy()
    kw = {}
    if history:                                                               # a presence penalty of 0.5 on some of the tokens first
        seen = np.stack([ids[rng.integers(0, n, 40)] for ids, _ in lists])
        kw = dict(history=torch.from_numpy(seen).cuda(), presence_penalty=0.5)
        for r in range(3):
            want[r, np.unique(seen[r])] -= np.float32(0.5)
    want = np.stack([added(want[r], *lists[r]) for r in range(3)])
    x = torch.from_numpy(z).cuda()
    got = lm.process_logits(x, bias_ids=torch.from_numpy(np.stack([i for i, _ in lists])).cuda(), bias_values=torch.from_numpy(np.stack([v for _, v in lists])).cuda(),
                            out=x if place == "same" else None, **kw)
    assert np.array_equal(got.cpu().numpy().view(np.int32), want.view(np.int32))


def test_repeated_entries_cost_no_square():
    """The longest list of one token, or filled up with one, is some 8000 dependent additions, a few hundred microseconds; walks by every entry were a third of a second. Lists of
    distinct tokens take 10 to 20 us: the limit is a thousand times that, a tenth of what the square cost."""
    rng = np.random.default_rng(0)
    n, vocab = 8191, 151_936
    x = torch.zeros(2, vocab, device="cuda", dtype=torch.bfloat16)

    def fastest(ids, values):
        ids, values = (torch.from_numpy(np.stack([t, t])).cuda() for t in (ids, values))
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            lm.process_logits(x, bias_ids=ids, bias_values=values)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    once = fastest(rng.permutation(vocab)[:n].astype(np.int32), np.zeros(n, dtype=np.float32))
    for kind in ("equal", "padded", "twice"):
        assert fastest(*repeated(rng, kind, vocab, n)) < 1000 * once


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shards_of_a_vocabulary(dtype):
    """Ids less a shard's first index, masks as views of whole words where it is a multiple of 32: the shards' results are the whole's columns."""
    rng = np.random.default_rng(5)
    rows, vocab = 5, 20_011
    x = torch.from_numpy((rng.standard_normal((rows, vocab)) * 3).astype(np.float32)).cuda().to(dtype)
    history = torch.from_numpy(rng.integers(-1, vocab + 3, (rows, 500)).astype(np.int32)).cuda()
    history[:, 0] = -2 ** 31
    ids = torch.from_numpy(rng.integers(-1, vocab, (rows, 60)).astype(np.int32)).cuda()
    kw = dict(repetition_penalty=1.25, presence_penalty=0.5, frequency_penalty=0.25, bias_values=torch.from_numpy(rng.normal(0, 4, (rows, 60)).astype(np.float32)).cuda())
    mask = torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32)).astype(np.int32)).cuda()
    bits = torch.int16 if dtype == torch.bfloat16 else torch.int32
    for cuts, masks in (([0, 7, 5000, 12_345, vocab], None), ([0, 32, 4992, 16_000, vocab], mask)):
        whole = lm.process_logits(x, history=history, bias_ids=ids, mask=masks, **kw)
        for lo, hi in zip(cuts[:-1], cuts[1:]):
            part = lm.process_logits(x[:, lo:hi], history=history - lo, bias_ids=ids - lo, mask=None if masks is None else masks[:, lo // 32:], **kw)
            assert torch.equal(part.view(bits), whole[:, lo:hi].contiguous().view(bits))
