"""The logits' processing on the GPU against its restatement in binary64 (oracle/logits.py). Logits that nothing names keep their bits, masked ones are -inf, the others lie within the
roundings of binary32 that the restatement counts and the last one (half a step: 2^-24 of the value in FP32, 2^-8 in BF16)."""
import numpy as np
import pytest
import torch

import lithos_metal_b200 as lm
import oracle
from oracle import logits as o

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BITS = {torch.float32: torch.int32, torch.bfloat16: torch.int16}


def cuda(x, dtype=None):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda() if dtype is None else torch.from_numpy(np.ascontiguousarray(x)).cuda().to(dtype)


def pack(allowed):
    rows, vocab = allowed.shape
    words = np.zeros((rows, (vocab + 31) // 32 * 32), dtype=np.uint8)
    words[:, :vocab] = allowed
    return np.packbits(words, axis=1, bitorder="little").view(np.int32)


def make(rng, rows, vocab, hist=0, bias=0, mask="none", shared=False):
    """Arguments in numpy; ids of both ends of the vocabulary and outside it among them."""
    kw = {}
    if hist:
        h = (rng.random((1 if shared else rows, hist)) ** 3 * vocab).astype(np.int32)
        h[:, ::7] = rng.choice(np.array([-1, 0, vocab - 1, vocab, 2 ** 31 - 1, -2 ** 31], dtype=np.int32), h[:, ::7].shape)
        kw["history"] = np.repeat(h, rows, 0) if shared else h
        kw["history_len"] = rng.integers(0, hist + 1, rows).astype(np.int32)
        kw["history_len"][0] = 0
        kw["history_len"][-1] = hist + 5                                     # (limited to the buffer)
        kw["prompt_len"] = rng.integers(0, hist + 1, rows).astype(np.int32)
        kw["repetition"], kw["presence"], kw["frequency"] = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.4), (-0.5, 1.0), (0.0, 0.5)))
    if bias:
        ids = rng.integers(-2, vocab + 2, (rows, bias)).astype(np.int32)
        ids[:, bias // 2:] = ids[:, :bias - bias // 2][:, ::-1]                # every other one twice
        if hist:
            ids[:, 0] = kw["history"][:, 0]
        kw["bias_ids"], kw["bias_values"] = ids, rng.normal(0, 5, (rows, bias)).astype(np.float32)
    if mask != "none":
        n = rows if mask == "grammar" else 3
        kw["mask"] = pack(rng.random((n, vocab)) < rng.choice([0.02, 0.5, 0.98], (n, 1)))
        kw["mask"][:, : (vocab + 31) // 64] = np.where(rng.random((n, 1)) < 0.5, kw["mask"][:, : (vocab + 31) // 64], rng.choice([0, -1], (n, (vocab + 31) // 64))).astype(np.int32)
        if mask == "rows":
            kw["mask"][0] = 0                                                # nothing allowed
            kw["mask_rows"] = rng.integers(-1, 4, rows).astype(np.int32)         # -1: none, 3: no such mask
            kw["mask_rows"][0] = 0
    return kw


def on_gpu(kw):
    names = dict(repetition="repetition_penalty", presence="presence_penalty", frequency="frequency_penalty")
    return {names.get(k, k): cuda(v) for k, v in kw.items()}


def logits_of(rng, rows, vocab, dtype):
    z = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    z[:, : min(vocab, 4)] = [[0.0, -0.0, np.inf, -np.inf][: min(vocab, 4)]]
    return cuda(z, dtype)


def check(got, before, kw, dtype):
    z = before.float().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want, bound, touched = o.process(z, **kw)
    have = got.float().cpu().numpy().astype(np.float64)
    hidden = np.isneginf(want) & ~np.isneginf(z)
    assert np.isneginf(have[hidden]).all()
    same = ~touched & ~(np.isneginf(want) & (kw.get("mask") is not None))
    a, b = got.view(BITS[dtype]).cpu().numpy(), before.view(BITS[dtype]).cpu().numpy()
    assert np.array_equal(a[same], b[same])
    finite = touched & np.isfinite(want)
    limit = bound + HALF[dtype] * (np.abs(want) + bound) + 1e-44
    assert (np.abs(have[finite] - want[finite]) <= limit[finite]).all()
    odd = touched & ~np.isfinite(want)
    assert np.array_equal(have[odd], want[odd], equal_nan=True)


SHAPES = [(1, 1), (1, 33), (3, 1000), (5, 4099), (2, 151936), (40, 20011)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("what", ["nothing", "history", "bias", "mask", "rows", "all"])
def test_against_the_definition(rows, vocab, what, dtype):
    rng = np.random.default_rng(rows * 31 + vocab + len(what))
    kw = make(rng, rows, vocab, hist=200 if what in ("history", "all") else 0, bias=40 if what in ("bias", "all") else 0,
              mask={"mask": "grammar", "rows": "rows", "all": "rows"}.get(what, "none"))
    x = logits_of(rng, rows, vocab, dtype)
    before = x.clone()
    got = lm.process_logits(x, **on_gpu(kw))
    assert torch.equal(x.view(BITS[dtype]), before.view(BITS[dtype])) and got.data_ptr() != x.data_ptr()
    check(got, before, kw, dtype)
    place = lm.process_logits(x, **on_gpu(kw), out=x)                         # in place
    assert place.data_ptr() == x.data_ptr() and torch.equal(x.view(BITS[dtype]), got.view(BITS[dtype]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_at_any_address(dtype):
    rng = np.random.default_rng(1)
    rows, vocab = 9, 3001
    kw = make(rng, rows, vocab, 64, 20, "rows")
    for at_in, at_out, width in ((0, 0, 3001), (1, 1, 3007), (3, 6, 3013), (8, 5, 3016)):
        wide, out = torch.zeros(rows, width + 16, dtype=dtype, device="cuda"), torch.full((rows + 2, width + 16), 5.0, dtype=dtype, device="cuda")
        wide[:, at_in:at_in + vocab] = logits_of(rng, rows, vocab, dtype)
        view = wide[:, at_in:at_in + vocab]
        check(lm.process_logits(view, **on_gpu(kw), out=out[1:-1, at_out:at_out + vocab]), view.clone(), kw, dtype)
        assert (out[0] == 5).all() and (out[-1] == 5).all() and (out[:, :at_out] == 5).all() and (out[:, at_out + vocab:] == 5).all()
    # two halves of one matrix; every other row; rows one after the other in reverse order are copied
    wide = torch.zeros(rows, 2 * vocab, dtype=dtype, device="cuda")
    wide[:, :vocab] = logits_of(rng, rows, vocab, dtype)
    check(lm.process_logits(wide[:, :vocab], **on_gpu(kw), out=wide[:, vocab:]), wide[:, :vocab].clone(), kw, dtype)
    many = logits_of(rng, 2 * rows, vocab, dtype)
    check(lm.process_logits(many[::2], **on_gpu(kw)), many[::2].clone(), kw, dtype)
    check(lm.process_logits(many[0].expand(rows, vocab), **on_gpu(kw)), many[0].expand(rows, vocab).clone(), kw, dtype)


@pytest.mark.parametrize("rows,vocab", [(8, 151936), (300, 5003), (1500, 1000)])
def test_long_histories_and_many_rows(rows, vocab):
    rng = np.random.default_rng(rows)
    kw = make(rng, rows, vocab, 5000 if rows < 100 else 300, 0, "rows")
    x = logits_of(rng, rows, vocab, torch.bfloat16)
    check(lm.process_logits(x, **on_gpu(kw)), x, kw, torch.bfloat16)


def test_the_longest_lists():
    rng = np.random.default_rng(8)
    history = np.full((2, 65536), 77, dtype=np.int32)
    history[1] = rng.integers(0, 1000, 65536)
    ids = np.concatenate([np.full(4000, 5), rng.integers(0, 1000, 4191)]).astype(np.int32)
    values = rng.integers(-8, 9, 8191).astype(np.float32)                     # (integers: the sums are exact)
    kw = dict(history=history, repetition=np.float32(1.1), presence=np.float32(0.25), frequency=np.float32(0.5), bias_ids=np.stack([ids] * 2), bias_values=np.stack([values] * 2))
    x = logits_of(rng, 2, 1000, torch.float32)
    got = lm.process_logits(x, history=cuda(history), repetition_penalty=1.1, presence_penalty=0.25, frequency_penalty=0.5, bias_ids=cuda(ids), bias_values=cuda(values))
    check(got, x, kw, torch.float32)
    with pytest.raises(lm._lib.LithosError):
        lm.process_logits(x, history=cuda(np.zeros((2, 65537), dtype=np.int32)))
    with pytest.raises(lm._lib.LithosError):
        lm.process_logits(x, bias_ids=cuda(np.zeros((2, 8192), dtype=np.int32)), bias_values=cuda(np.zeros((2, 8192), dtype=np.float32)))


def test_biases_of_one_token_are_added_in_list_order():
    values = np.array([[1e8, 1.0, -1e8, 3.0], [1.0, 1e8, -1e8, 3.0]], dtype=np.float32)
    ids = np.full((2, 4), 6, dtype=np.int32)
    ids[:, 3] = -1
    x = torch.zeros(2, 10, device="cuda")
    got = lm.process_logits(x, bias_ids=cuda(ids), bias_values=cuda(values))
    want = [[np.float32(np.float32(np.float32(1e8) + 1) - np.float32(1e8))], [np.float32(np.float32(np.float32(1.0) + np.float32(1e8)) - np.float32(1e8))]]
    assert got[:, 6].cpu().tolist() == [w[0] for w in want] and got.count_nonzero() <= 2
    inf = lm.process_logits(x, bias_ids=cuda(ids), bias_values=cuda(np.array([[-np.inf, 1, 1, 1]] * 2, dtype=np.float32)))
    assert torch.isneginf(inf[:, 6]).all()


def test_infinities_and_nan_behind_a_mask():
    x = torch.tensor([[float("nan"), float("inf"), -float("inf"), 1.0, torch.finfo(torch.bfloat16).min, 2.0, 3.0, 4.0, 5.0]] * 2, dtype=torch.bfloat16, device="cuda")
    mask = pack(np.array([[0, 0, 0, 1, 1, 0, 1, 1, 1], [1, 1, 1, 1, 1, 1, 1, 1, 0]], dtype=bool))
    history = np.array([[0, 1, 2, 3, 4, 8]] * 2, dtype=np.int32)
    got = lm.process_logits(x, mask=cuda(mask), history=cuda(history), repetition_penalty=2.0).float().cpu().numpy()
    assert np.isneginf(got[0, [0, 1, 2, 5]]).all() and got[0, 3] == 0.5 and np.isneginf(got[0, 4]) and got[0, 6:].tolist() == [3.0, 4.0, 2.5]
    assert np.isnan(got[1, 0]) and got[1, 1] == np.inf and np.isneginf(got[1, 2]) and got[1, 3] == 0.5 and got[1, 5] == 2.0 and np.isneginf(got[1, 8])


@pytest.mark.parametrize("history", [False, True])
def test_rows_with_masks_that_do_not_exist(history):
    """mask_rows beyond the masks hides the whole row, none at all included; a negative one leaves it alone."""
    x = torch.randn(3, 500, device="cuda")
    rows = torch.tensor([-1, 0, 7], dtype=torch.int32, device="cuda")
    kw = dict(history=torch.zeros(3, 1, dtype=torch.int32, device="cuda")) if history else {}
    for masks in (0, 1):
        mask = torch.full((masks, 16), -1, dtype=torch.int32, device="cuda")
        for m, r in ((mask, rows), (mask, rows.long())):                     # (as it is, and converted)
            got = lm.process_logits(x, mask=m, mask_rows=r, **kw)
            assert torch.equal(got[0], x[0]) and torch.isneginf(got[2]).all()
            assert torch.equal(got[1], x[1]) if masks else torch.isneginf(got[1]).all()


def test_plain_penalties_are_the_samplers():
    """With numbers, no prompt and no frequency, processing and then sampling FP32 logits is sampling with that history."""
    rng = np.random.default_rng(12)
    rows, vocab = 6, 40000
    x = cuda((rng.standard_normal((rows, vocab)) * 2).astype(np.float32))
    history = cuda(rng.integers(0, vocab, (rows, 500)).astype(np.int32))
    u = cuda(rng.random(rows).astype(np.float32))
    knobs = dict(temperature=0.8, top_k=50, top_p=0.9, draw="inverse_cdf")
    a = lm.sample(x, lm.SamplingParams(**knobs, repetition_penalty=1.3, presence_penalty=0.7), history=history, uniforms=u, return_tau=True)
    y = lm.process_logits(x, history=history, repetition_penalty=1.3, presence_penalty=0.7)
    b = lm.sample(y, lm.SamplingParams(**knobs), uniforms=u, return_tau=True)
    assert torch.equal(a.tokens, b.tokens) and torch.equal(a.tau, b.tau)


def test_the_rows_of_a_speculative_round():
    """One buffer of tokens for all rows, longer by a draft from row to row (row stride 0), numbers and tensors mixed."""
    rng = np.random.default_rng(13)
    rows, vocab, n = 8, 50264, 120
    h = rng.integers(0, 3000, n).astype(np.int32)
    lens = np.arange(n - rows + 1, n + 1).astype(np.int32)
    x = logits_of(rng, rows, vocab, torch.bfloat16)
    kw = dict(history=np.stack([h] * rows), history_len=lens, repetition=np.full(rows, 1.2, np.float32), presence=np.float32(0.0), frequency=np.float32(0.25))
    for history in (cuda(h), cuda(h).expand(rows, n)):
        got = lm.process_logits(x, history=history, history_len=cuda(lens), repetition_penalty=torch.full((rows,), 1.2, device="cuda"), frequency_penalty=0.25)
        check(got, x, kw, torch.bfloat16)


def test_conversions_of_the_arguments():
    """int64 ids on the host, float64 knobs, a mask wider than the vocabulary: converted, with the same result."""
    rng = np.random.default_rng(14)
    kw = make(rng, 4, 777, 30, 10, "grammar")
    x = logits_of(rng, 4, 777, torch.float32)
    want = lm.process_logits(x, **on_gpu(kw))
    wide = torch.zeros(4, 40, dtype=torch.int32, device="cuda")
    wide[:, : kw["mask"].shape[1]] = cuda(kw["mask"])
    got = lm.process_logits(x, history=torch.from_numpy(kw["history"]), history_len=torch.from_numpy(kw["history_len"]).long(), prompt_len=cuda(kw["prompt_len"]).long(),
                            repetition_penalty=cuda(kw["repetition"]).double(), presence_penalty=cuda(kw["presence"]), frequency_penalty=torch.from_numpy(kw["frequency"]),
                            bias_ids=cuda(kw["bias_ids"]).long(), bias_values=cuda(kw["bias_values"]).double(), mask=wide)
    assert torch.equal(got.view(torch.int32), want.view(torch.int32))
    t = lm.process_logits(x.T.contiguous().T, **on_gpu(kw))
    assert torch.equal(t.view(torch.int32), want.view(torch.int32))


def test_offsets_past_32_bits():
    """4400 rows of 1,048,576 logits: the last rows are those of a call of their own, into another place and in place."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    rows, vocab = 4400, 1 << 20
    x = torch.randn(64, vocab, device="cuda", generator=gen).bfloat16().repeat(70, 1)[:rows]
    history = torch.randint(0, vocab, (rows, 100), device="cuda", generator=gen, dtype=torch.int32)
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, vocab // 32), device="cuda", generator=gen, dtype=torch.int32)
    for kw in (dict(history=history), dict(mask=mask), dict(history=history, mask=mask)):
        want = lm.process_logits(x[-3:], repetition_penalty=1.3, **{k: v[-3:] for k, v in kw.items()}).view(torch.int16)
        assert torch.equal(lm.process_logits(x, repetition_penalty=1.3, **kw)[-3:].view(torch.int16), want)
        place = x.clone()
        assert torch.equal(lm.process_logits(place, repetition_penalty=1.3, out=place, **kw)[-3:].view(torch.int16), want)


def test_refusals():
    x = torch.zeros(3, 100, device="cuda")
    ids = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    bad = [dict(history=ids[:2]), dict(history=ids, history_len=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(bias_ids=ids), dict(bias_values=ids.float()),
           dict(bias_ids=ids, bias_values=ids[:, :3].float()), dict(mask=torch.zeros(3, 3, dtype=torch.int32, device="cuda")), dict(mask=torch.zeros(2, 4, dtype=torch.int32, device="cuda")),
           dict(mask=torch.zeros(3, 4, dtype=torch.int64, device="cuda")), dict(mask_rows=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(repetition_penalty=0.0, history=ids),
           dict(repetition_penalty=torch.ones(2, device="cuda"), history=ids), dict(out=torch.zeros(3, 101, device="cuda")), dict(out=torch.zeros(3, 100, dtype=torch.bfloat16, device="cuda"))]
    for kw in bad:
        with pytest.raises(ValueError):
            lm.process_logits(x, **kw)
    with pytest.raises(TypeError):
        lm.process_logits(x.half())
    with pytest.raises(RuntimeError):
        lm.process_logits(x.cpu())
    with pytest.raises(ValueError):                                          # in place wants rows that lie together
        t = torch.zeros(100, 3, device="cuda").T
        lm.process_logits(t, out=t)
    buffer = torch.zeros(4, 100, device="cuda")
    for view, out in ((buffer[:3], buffer[1:]), (buffer.view(-1)[:300].view(3, 100), buffer.view(-1)[50:350].view(3, 100))):   # that overlap
        with pytest.raises(lm._lib.LithosError):
            lm.process_logits(view, out=out)
    assert lm.process_logits(x[:0]).shape == (0, 100) and lm.process_logits(x[:, :0]).shape == (3, 0)


def test_captured_and_on_another_stream():
    rng = np.random.default_rng(15)
    kw = on_gpu(make(rng, 20, 9000, 100, 10, "rows"))
    x = logits_of(rng, 20, 9000, torch.bfloat16)
    want = lm.process_logits(x, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lm.process_logits(x, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other.view(torch.int16), want.view(torch.int16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lm.process_logits(x, **kw)
    kw["history"].random_(0, 9000)
    kw["presence_penalty"].mul_(2.0)
    graph.replay()
    assert torch.equal(out.view(torch.int16), lm.process_logits(x, **kw).view(torch.int16))


@pytest.mark.parametrize("rows", [1, 8, 40])
def test_the_decode_tail(rows):
    """4-bit projection, processing under a grammar, thresholds and draw: the sampler's tokens are the oracle's on the processed logits and allowed by the mask, drawn and greedy."""
    rng = np.random.default_rng(16)
    hidden, vocab = 512, 32768
    w = lm.quantize_nvfp4(cuda((rng.standard_normal((vocab, hidden)) * 0.05).astype(np.float32)))
    x = cuda(rng.standard_normal((rows, hidden)).astype(np.float32), torch.bfloat16)
    kw = make(rng, rows, vocab, 100, 8, "none")
    allowed = rng.random((rows, vocab)) < 0.01
    allowed[0] = False
    allowed[0, 321] = True                                                   # one token only
    logits = lm.lm_head(x, w)
    lm.process_logits(logits, **on_gpu(kw), mask=cuda(pack(allowed)), out=logits)
    u = rng.random(rows).astype(np.float32)
    codes = logits.view(torch.int16).cpu().numpy().view(np.uint16)
    for knobs in (dict(temperature=0.8, top_k=50, top_p=0.95), dict(temperature=1.0, top_p=0.9), dict(temperature=0.0)):
        r = lm.sample(logits, lm.SamplingParams(**knobs, draw="inverse_cdf"), uniforms=cuda(u))
        tok, _, _ = oracle.sample_batch(codes, draw="inverse_cdf", uniforms=u, n_threads=8, **knobs)
        assert r.tokens.cpu().tolist() == tok.tolist() and allowed[np.arange(rows), tok].all()
    assert torch.equal(lm.argmax(logits).cpu(), torch.from_numpy(codes.view(np.int16)).view(torch.bfloat16).float().argmax(-1).to(torch.int32))
