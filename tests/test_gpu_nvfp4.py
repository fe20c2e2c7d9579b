"""The microscaled 4-bit weight and the projection with it on the GPU, against the binary64 restatement (oracle/nvfp4.py). Codes and block scales are equal, bit for
bit: they are defined as roundings of real quotients. A logit is the BF16 rounding (half a step: 2^-8 of the value) of a sum whose FP32 accumulation may be off by
2^-23 of the magnitudes' sum per addition."""
import copy
import threading

import numpy as np
import pytest
import torch

import lithos_metal_b200 as lm
import oracle
from oracle import head as o_head
from oracle import nvfp4 as o

pytestmark = pytest.mark.gpu


def bf16(codes):
    return torch.from_numpy(np.ascontiguousarray(codes).view(np.int16)).cuda().view(torch.bfloat16)


def quantized(x, scale=None):
    w = lm.quantize_nvfp4(x, scale=scale)
    return w, w.codes.cpu().numpy(), w.scales.cpu().numpy(), np.float32(w.scale.item())


def random_weight(rng, vocab, hidden, g=0.01):
    """Any codes and any finite positive scales: what a checkpoint could hold."""
    codes = rng.integers(0, 256, (vocab, hidden // 2), dtype=np.uint8)
    scales = rng.integers(0, 127, (vocab, hidden // 16)).astype(np.uint8)
    return codes, scales, np.float32(g)


def as_weight(codes, scales, g):
    return lm.Nvfp4Weight(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), torch.tensor([g], dtype=torch.float32, device="cuda"))


def check_head(got, x, codes, scales, g, extra=0.0):
    want, bound = o.head(x, codes, scales, g)
    bound = bound + extra
    error = np.abs(got.float().cpu().numpy().astype(np.float64) - want)
    limit = bound + 2.0 ** -8 * (np.abs(want) + bound)
    assert (error <= limit).all(), float((error / np.maximum(limit, 1e-300)).max())


# ---- the format -----------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 48), (257, 1040), (64, 4096)])
def test_codes_are_the_definitions(rows, cols, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=gen, device="cuda") * 0.03 * torch.exp(2.0 * torch.randn(rows, 1, generator=gen, device="cuda"))).to(dtype)
    w, codes, scales, g = quantized(x)
    host = x.float().cpu().numpy()
    assert g == o.global_scale(host)
    want_codes, want_scales = o.quantize(host, g)
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)
    assert np.array_equal(w.dequantize().cpu().numpy(), (o.values(codes, scales, np.float32(1.0)).astype(np.float32) * g))
    given = torch.tensor([float(g) * 1.7], dtype=torch.float32, device="cuda")
    _, codes, scales, g2 = quantized(x, given)
    want_codes, want_scales = o.quantize(host, g2)
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)


@pytest.mark.parametrize("g", [1.0, 2.0 ** -7, 0.3, 2.0 ** -120, 2.0 ** 110])
def test_every_border_and_its_neighbours(g):
    """Inputs on, just below and just above every border between two codes, and every border between two block scales."""
    g = np.float32(g)
    rng = np.random.default_rng(7)
    blocks = []
    for s in list(range(1, 127, 5)) + [126]:
        unit = o.E4M3[s] * np.float64(g)
        for border in (o.E2M1[:-1] + o.E2M1[1:]) / 2:
            v = np.float32(border * unit)
            b = np.zeros(16, dtype=np.float32)
            b[0] = np.float32(6 * unit)                                      # keeps the block's scale where it is
            b[1:4] = [np.nextafter(v, np.float32(0)), v, np.nextafter(v, np.float32(np.inf))]
            b[4:7] = -b[1:4]
            blocks.append(b)
    for lo, hi in zip(o.E4M3[:-1], o.E4M3[1:]):
        v = np.float32((lo + hi) / 2 * 6.0 * np.float64(g))
        for a in (np.nextafter(v, np.float32(0)), v, np.nextafter(v, np.float32(np.inf))):
            b = (rng.standard_normal(16) * 0.2 * a).astype(np.float32).clip(-a, a)
            b[5] = -a
            blocks.append(b)
    x = np.stack(blocks)
    _, codes, scales, _ = quantized(torch.from_numpy(x).cuda(), torch.tensor([g], device="cuda"))
    want_codes, want_scales = o.quantize(x, g)
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)


@pytest.mark.parametrize("g", [0.0, -0.0, -1.0, float("inf"), float("nan"), 1e-40, 1e-45, 3e38])
def test_a_scale_of_any_kind(g):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((8, 64)).astype(np.float32)
    x[0, 0], x[1, :16], x[2, 3], x[3, 20] = 0.0, 0.0, np.inf, np.nan
    _, codes, scales, _ = quantized(torch.from_numpy(x).cuda(), torch.tensor([g], device="cuda"))
    with np.errstate(all="ignore"):
        want_codes, want_scales = o.quantize(x, np.float32(g))
    assert np.array_equal(codes, want_codes) and np.array_equal(scales, want_scales)


def test_zeros_infinities_and_nan():
    x = np.zeros((6, 64), dtype=np.float32)
    x[1, 3], x[2, 20], x[3, 40] = np.inf, np.nan, -np.inf
    x[1:4, 63] = 1.5
    x[4] = -0.0
    x[5, :16] = 1e-20                                                        # far below the block scale of the largest: scale 0
    w, codes, scales, g = quantized(torch.from_numpy(x).cuda())
    want_codes, want_scales = o.quantize(x, g)
    assert g == np.float32(1.5) / np.float32(2688) and np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)
    v = w.dequantize().cpu().numpy()
    assert np.isnan(v[1, :16]).all() and np.isnan(v[2, 16:32]).all() and np.isnan(v[3, 32:48]).all() and np.isfinite(v[[0, 4, 5]]).all()
    assert v[1, 63] == np.float32(2688.0) * g        # (code 6, scale 448: 2688 times fl32(1.5 / 2688), two roundings from 1.5: up to 2^-23 of it away)
    # nothing but zeros, an empty matrix, and scales that are none
    w, codes, scales, g = quantized(torch.zeros(2, 32, device="cuda"))
    assert g == 1.0 and not codes.any() and not scales.any()
    assert lm.quantize_nvfp4(torch.zeros(0, 32, device="cuda")).dequantize().shape == (0, 32)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        _, codes, scales, _ = quantized(torch.ones(1, 16, device="cuda"), torch.tensor([bad], device="cuda"))
        assert scales.tolist() == [[127]] and not codes.any()


def test_strides_of_a_view():
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(40, 200, generator=gen, device="cuda")
    for x in (wide[:, 3:3 + 96], wide[::2, 8:8 + 96], wide.bfloat16()[:, 5:5 + 96], wide[:, :96].T.contiguous().T[:, :96]):
        _, codes, scales, g = quantized(x)
        want_codes, want_scales = o.quantize(x.float().cpu().numpy(), g)
        assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)
    w = lm.quantize_nvfp4(wide[:, :96].contiguous())
    out = torch.full((40, 101), 7.0, device="cuda")
    w.dequantize(out=out[:, 3:99])
    assert torch.equal(out[:, 3:99], w.dequantize()) and (out[:, :3] == 7).all() and (out[:, 99:] == 7).all()
    part = w[10:25]
    assert part.shape == (15, 96) and torch.equal(part.dequantize(), w.dequantize()[10:25])


# ---- the projection ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 33, 64, 100, 129, 256, 300])
@pytest.mark.parametrize("hidden,vocab", [(64, 17), (192, 1000), (1024, 4099)])
def test_head_against_the_definition(rows, hidden, vocab):
    rng = np.random.default_rng(rows * 7 + vocab)
    codes, scales, g = random_weight(rng, vocab, hidden)
    x = bf16(oracle.f32_to_bf16((rng.standard_normal((rows, hidden)) * np.exp(rng.standard_normal((rows, 1)) * 3)).astype(np.float32)))
    got = lm.lm_head(x, as_weight(codes, scales, g))
    assert got.shape == (rows, vocab) and got.dtype == torch.bfloat16
    check_head(got, x.float().cpu().numpy(), codes, scales, g)


@pytest.mark.parametrize("rows", [1, 5, 8, 20, 130])
@pytest.mark.parametrize("one_plus", [True, False])
def test_head_with_the_norm_fused(rows, one_plus):
    rng = np.random.default_rng(rows)
    hidden, vocab, eps = 2048, 3001, 1e-5
    codes, scales, g = random_weight(rng, vocab, hidden)
    x = oracle.f32_to_bf16((rng.standard_normal((rows, hidden)) * 2).astype(np.float32))
    gamma = oracle.f32_to_bf16((rng.standard_normal(hidden) * 0.1).astype(np.float32))
    got = lm.lm_head(bf16(x), as_weight(codes, scales, g), bf16(gamma), eps=eps, one_plus=one_plus)
    # The norm's output is rounded to BF16: where the binary64 value lies next to a midpoint the FP32 one may round to its other neighbour. In FP32 some 21 roundings lie in a sum of
    # squares (8 of a thread's, the joining), 2 in the mean and eps, all under the root (half of each), then the root, 1 + weight and two products: less than 16 * 2^-24 in all.
    xf, gf = o_head._f32(x).astype(np.float64), o_head._f32(gamma).astype(np.float64)
    y = xf / np.sqrt((xf * xf).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * ((1.0 + gf) if one_plus else gf)
    near = 2.0 ** -20 * np.abs(y)
    lo, hi = (o_head._f32(o_head._bf16((y + d).astype(np.float32))).astype(np.float64) for d in (-near, near))
    w = np.abs(o.values(codes, scales, g))
    check_head(got, lo, codes, scales, g, extra=np.abs(hi - lo) @ w.T)


@pytest.mark.parametrize("rows", [1, 8, 40, 200])
def test_values_of_any_size_in_x(rows):
    """Elements of a row further apart than binary16 reaches, subnormal rows, zero rows: the products are exact all the same."""
    rng = np.random.default_rng(11 + rows)
    hidden, vocab = 256, 300
    codes, scales, g = random_weight(rng, vocab, hidden, 2.0 ** -9)
    x = (rng.standard_normal((rows, hidden)) * 2.0 ** rng.integers(-60, 40, (rows, hidden))).astype(np.float32)
    x[0] = 0.0
    if rows > 4:
        x[2] = rng.standard_normal(hidden).astype(np.float32) * 1e-39          # BF16 subnormals
        x[3, :] = 0.0
        x[3, 7], x[3, 100] = 3e37, 1e-30
        x[4] = rng.standard_normal(hidden).astype(np.float32)
    t = bf16(oracle.f32_to_bf16(x))
    got = lm.lm_head(t, as_weight(codes, scales, g))
    host = t.float().cpu().numpy().astype(np.float64)
    want, bound = o.head(host, codes, scales, g)
    error = np.abs(got.float().cpu().numpy().astype(np.float64) - want)
    limit = bound + 2.0 ** -8 * (np.abs(want) + bound) + 2.0 ** -133           # (and half a BF16 subnormal step)
    limit[np.abs(want) > 3.0e38] = np.inf                                    # (beyond BF16)
    assert (error <= limit).all() and (got[0] == 0).all()
    # a row with infinities or NaN does not reach the other rows
    t2 = t.clone()
    t2[-1, 5] = float("inf")
    t2[-1, 9] = float("nan")
    again = lm.lm_head(t2, as_weight(codes, scales, g))
    assert torch.isnan(again[-1]).all()
    if rows > 1:
        e2 = np.abs(again[:-1].float().cpu().numpy().astype(np.float64) - want[:-1])
        assert (e2 <= limit[:-1]).all()


@pytest.mark.parametrize("rows", [1, 3, 9])
@pytest.mark.parametrize("small", [1e-7, 1e-9, 1e-20, 1e-30, 1e-39])
def test_a_small_element_beside_a_large_one(rows, small):
    """Where the large element's code is 0 the small one's product is the whole logit."""
    rng = np.random.default_rng(3)
    codes, scales, g = random_weight(rng, 200, 64, 2.0 ** -6)
    codes[::2, 3] &= 0xF8                                                   # column 6: magnitude 0 in every other row
    x = np.zeros((rows, 64), dtype=np.float32)
    x[:, 6], x[:, 33] = 1e6, small
    t = bf16(oracle.f32_to_bf16(x))
    want, bound = o.head(t.float().cpu().numpy(), codes, scales, g)
    error = np.abs(lm.lm_head(t, as_weight(codes, scales, g)).float().cpu().numpy().astype(np.float64) - want)
    assert (error <= bound + 2.0 ** -8 * (np.abs(want) + bound) + 2.0 ** -134).all()      # (2^-134: half a BF16 subnormal step)


@pytest.mark.parametrize("rows", [1, 8, 24, 140])
def test_a_nan_scale_reaches_its_row_of_the_weight_only(rows):
    rng = np.random.default_rng(2)
    codes, scales, g = random_weight(rng, 90, 128)
    x = bf16(oracle.f32_to_bf16(rng.standard_normal((rows, 128)).astype(np.float32)))
    whole = lm.lm_head(x, as_weight(codes, scales, g))
    scales[33, 2] = 127
    got = lm.lm_head(x, as_weight(codes, scales, g))
    assert torch.isnan(got[:, 33]).all()
    keep = torch.arange(90, device="cuda") != 33
    assert torch.equal(got[:, keep].view(torch.int16), whole[:, keep].view(torch.int16))
    # negative scales are numbers too
    scales[33, 2] = 0x80 | 50
    check_head(lm.lm_head(x, as_weight(codes, scales, g)), x.float().cpu().numpy(), codes, scales, g)


@pytest.mark.parametrize("rows", [1, 8, 30, 256])
def test_a_shard_of_the_weight_gives_the_bits_of_the_whole(rows):
    rng = np.random.default_rng(9)
    codes, scales, g = random_weight(rng, 9000, 512)
    w = as_weight(codes, scales, g)
    x = bf16(oracle.f32_to_bf16(rng.standard_normal((rows, 512)).astype(np.float32)))
    whole = lm.lm_head(x, w)
    for shards in (2, 3, 8):
        parts = [lm.lm_head(x, w[lo:lo + width]) for lo, width in (lm.parallel.shard_vocab(9000, s, shards) for s in range(shards))]
        assert torch.equal(torch.cat(parts, dim=1).view(torch.int16), whole.view(torch.int16))


@pytest.mark.parametrize("rows,hidden,vocab", [(256, 4096, 20000), (200, 2048, 40000), (130, 4096, 20000), (128, 4096, 40000), (40, 4096, 40000), (17, 6400, 20000)])
def test_rows_together_are_the_rows_one_by_eight(rows, hidden, vocab):
    """Long runs of tiles and steps through every place of the batch kernel's shared memory, several times: within one BF16 unit of the few-rows kernel everywhere (two summation orders)."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    w = lm.Nvfp4Weight(torch.randint(0, 256, (vocab, hidden // 2), dtype=torch.uint8, device="cuda", generator=gen),
                       torch.randint(100, 120, (vocab, hidden // 16), dtype=torch.uint8, device="cuda", generator=gen), torch.tensor([0.001], device="cuda"))
    x = torch.randn(rows, hidden, device="cuda", generator=gen).bfloat16()
    want = torch.cat([lm.lm_head(x[r:r + 8], w) for r in range(0, rows, 8)])
    # sums of `hidden` products off by 2^-23 of the magnitudes' sum per addition on either side (means: |x| 0.8, the weight 0.273; the largest row's sum a quarter above that), two BF16 roundings
    close = 2 * (hidden * 2.0 ** -23) * (hidden * 0.8 * 0.273 * 1.25) + 2 * 2.0 ** -8 * want.float().abs()
    first = lm.lm_head(x, w)
    assert ((first.float() - want.float()).abs() <= close).all()
    for _ in range(6):
        assert torch.equal(lm.lm_head(x, w).view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("rows", [3, 8, 50, 256])
def test_strides_and_a_given_place(rows):
    rng = np.random.default_rng(4)
    codes, scales, g = random_weight(rng, 333, 192)
    wide_c, wide_s = torch.zeros(333, 96 + 32, dtype=torch.uint8, device="cuda"), torch.zeros(333, 16, dtype=torch.uint8, device="cuda")
    wide_c[:, 16:112], wide_s[:, 4:16] = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
    w = lm.Nvfp4Weight(wide_c[:, 16:112], wide_s[:, 4:16].view(torch.float8_e4m3fn), torch.tensor([g], device="cuda"))
    x = bf16(oracle.f32_to_bf16(rng.standard_normal((rows, 192 + 7)).astype(np.float32)))[:, 3:195]      # rows at odd addresses
    whole = lm.lm_head(x.contiguous(), as_weight(codes, scales, g))
    out = torch.full((rows + 2, 340), 7.0, dtype=torch.bfloat16, device="cuda")
    got = lm.lm_head(x, w, out=out[1:rows + 1, 5:338])
    assert got.data_ptr() == out[1:, 5:].data_ptr() and torch.equal(got.view(torch.int16), whole.view(torch.int16))
    assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[:, :5] == 7).all() and (out[:, 338:] == 7).all()
    assert lm.lm_head(x[:0], w).shape == (0, 333) and lm.lm_head(x, w[:0]).shape == (rows, 0)


@pytest.mark.parametrize("rows", [1, 16, 17, 70])
@pytest.mark.parametrize("hidden", [64, 320])
def test_one_row_of_the_weight(rows, hidden):
    """Its strides are of no account, aligned or not."""
    rng = np.random.default_rng(hidden + rows)
    codes, scales, g = random_weight(rng, 3, hidden)
    x = bf16(oracle.f32_to_bf16(rng.standard_normal((rows, hidden)).astype(np.float32)))
    for w in (as_weight(codes[1:2].copy(), scales[1:2].copy(), g), as_weight(codes, scales, g)[1:2]):
        got = lm.lm_head(x, w)
        assert got.shape == (rows, 1)
        check_head(got, x.float().cpu().numpy(), codes[1:2], scales[1:2], g)


def test_a_weight_keeps_its_tensors():
    w = lm.quantize_nvfp4(torch.ones(20, 64, device="cuda"))
    with pytest.raises(AttributeError):
        w.codes = w.codes[:3]
    again = copy.deepcopy(w)
    assert again.codes.data_ptr() != w.codes.data_ptr() and torch.equal(again.dequantize(), w.dequantize())
    again.codes.zero_()
    assert (again.dequantize() == 0).all() and (w.dequantize() != 0).all()


def test_two_threads_at_once():
    rng = np.random.default_rng(8)
    codes, scales, g = random_weight(rng, 30000, 512)
    w = as_weight(codes, scales, g)
    xs = [bf16(oracle.f32_to_bf16(rng.standard_normal((n, 512)).astype(np.float32))) for n in (5, 40, 200)]
    want = [lm.lm_head(x, w).view(torch.int16) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(lm.lm_head(xs[i], w).view(torch.int16), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 2, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("rows,hidden,vocab", [(1, 12736, 300), (8, 12736, 300), (9, 12736, 300), (16, 6400, 300), (70, 12736, 300), (65536, 64, 40)])
def test_the_largest_sizes(rows, hidden, vocab):
    gen = torch.Generator(device="cuda").manual_seed(rows + hidden)
    w = lm.quantize_nvfp4(torch.randn(vocab, hidden, device="cuda", generator=gen))
    x = torch.randn(rows, hidden, device="cuda", generator=gen).bfloat16()
    values = w.dequantize().double()
    want = x.double() @ values.T
    # sums of `hidden` products off by 2^-23 of the magnitudes' sum per addition, then one BF16 rounding
    bound = hidden * 2.0 ** -23 * (x.double().abs() @ values.abs().T)
    got = lm.lm_head(x, w).double()
    assert ((got - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()


def test_offsets_past_32_bits():
    """A weight of 1,048,000 x 8192 (8.6e9 elements, 4.3 GB of codes): its last rows as a weight of their own give the same bits."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(1024, 8192, device="cuda", generator=gen).bfloat16().repeat(1024, 1)[:1_048_000]
    w = lm.quantize_nvfp4(x)
    last = lm.quantize_nvfp4(x[-3000:], scale=w.scale)
    assert torch.equal(w.codes[-3000:], last.codes) and torch.equal(w.scales[-3000:], last.scales)
    del x
    for rows in (2, 40, 300):
        h = torch.randn(rows, 8192, device="cuda", generator=gen).bfloat16()
        assert torch.equal(lm.lm_head(h, w)[:, -3000:].contiguous().view(torch.int16), lm.lm_head(h, last).view(torch.int16))


def test_refusals():
    w = lm.quantize_nvfp4(torch.ones(20, 64, device="cuda"))
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        lm.quantize_nvfp4(torch.zeros(2, 24, device="cuda"))
    with pytest.raises(TypeError):
        lm.quantize_nvfp4(torch.zeros(2, 32, dtype=torch.float16, device="cuda"))
    with pytest.raises(RuntimeError):
        lm.quantize_nvfp4(torch.zeros(2, 32))
    with pytest.raises(ValueError):
        lm.quantize_nvfp4(torch.zeros(2, 32, device="cuda"), scale=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError):
        lm.lm_head(x.float(), w)
    with pytest.raises(ValueError):
        lm.lm_head(x[:, :32], w)
    with pytest.raises(ValueError):
        lm.lm_head(x, w, torch.ones(63, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        lm.lm_head(x, w, out=torch.zeros(2, 21, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        lm.Nvfp4Weight(w.codes, w.scales[:, :2], w.scale)
    with pytest.raises(ValueError):
        lm.Nvfp4Weight(w.codes.to(torch.int8), w.scales, w.scale)
    with pytest.raises(TypeError):
        w[3]
    for rows, hidden in ((65537, 64), (2, 12800)):                           # beyond the largest sizes
        with pytest.raises(lm._lib.LithosError):
            lm.lm_head(torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda"), lm.quantize_nvfp4(torch.ones(2, hidden, device="cuda")))
    with pytest.raises(lm._lib.LithosError):                                 # a hidden size that is no multiple of 64
        lm.lm_head(torch.zeros(2, 48, dtype=torch.bfloat16, device="cuda"), lm.quantize_nvfp4(torch.ones(20, 48, device="cuda")))
    with pytest.raises(lm._lib.LithosError):                                 # codes off their alignment
        c = torch.zeros(20 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(20, 32)
        lm.lm_head(x, lm.Nvfp4Weight(c, w.scales, w.scale))


def test_captured_replayed_and_on_another_stream():
    rng = np.random.default_rng(5)
    codes, scales, g = random_weight(rng, 5000, 256)
    w = as_weight(codes, scales, g)
    a, b = (bf16(oracle.f32_to_bf16(rng.standard_normal((n, 256)).astype(np.float32))) for n in (8, 70))
    want = [lm.lm_head(t, w).clone() for t in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [lm.lm_head(t, w) for t in (a, b)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, other))
    graphs, outs = [], []
    for t in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(lm.lm_head(t, lm.quantize_nvfp4(w.dequantize(), scale=w.scale)))
        graphs.append(graph)
    keep = [t.clone() for t in (a, b)]
    for t in (a, b):
        t.mul_(-1.0)
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):                                                       # both at once
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    again = lm.quantize_nvfp4(w.dequantize(), scale=w.scale)
    for t, out in zip(keep, outs):
        assert torch.equal(out, lm.lm_head(-t, again))
