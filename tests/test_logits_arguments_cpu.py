"""The conversions of the logits' processing's arguments without a GPU."""
import pytest
import torch

from lithos_metal_b200 import logits

CPU = torch.device("cpu")


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint64, torch.float64])
def test_wide_values_name_nothing_else(dtype):
    """Ids, lengths and rows of masks beyond int32 stay beyond every vocabulary, length and number of masks."""
    values = [0, 5, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 5, 2 ** 40 + 7]
    values += {torch.int64: [2 ** 63 - 1, -1, -2 ** 31 - 1, -2 ** 32 + 5, -2 ** 63], torch.uint64: [2 ** 63 - 1, 2 ** 63, 2 ** 63 + 5, 2 ** 64 - 1], torch.float64: [-1.0, -2.0 ** 32 + 5]}[dtype]
    want = [min(max(int(v), -2 ** 31), 2 ** 31 - 1) for v in values]
    t = torch.tensor(values, dtype=dtype)
    assert logits._rows_of(t, 2, torch.int32, CPU, "ids").tolist() == [want, want]
    assert logits._lengths(t, len(values), CPU, "lengths").tolist() == want


@pytest.mark.parametrize("dtype", [torch.int32, torch.int16, torch.int8, torch.uint8, torch.uint32])
def test_narrow_values_are_themselves(dtype):
    values = [0, 1, 100] + ([] if dtype in (torch.uint8, torch.uint32) else [-1])
    assert logits._rows_of(torch.tensor(values, dtype=dtype), 1, torch.int32, CPU, "ids").tolist() == [values]
    assert logits._lengths(torch.tensor([2 ** 32 - 1, 3], dtype=torch.uint32), 2, CPU, "lengths").tolist() == [2 ** 31 - 1, 3]
    given = torch.arange(6, dtype=torch.int32).view(2, 3)
    assert logits._rows_of(given, 2, torch.int32, CPU, "ids").data_ptr() == given.data_ptr()         # (as it is)
    assert logits._rows_of(torch.tensor([[1.5, 2.0 ** 33]], dtype=torch.float64), 1, torch.float32, CPU, "values").tolist() == [[1.5, 2.0 ** 33]]


@pytest.mark.gpu
def test_wide_values_on_the_gpu():
    x = torch.randn(2, 500, device="cuda")
    far = torch.tensor([[2 ** 32 + 5, -2 ** 32 + 6, 7]] * 2)
    want = x.clone()
    want[:, 7] += 1.0
    for ids in (far, far.cuda()):
        assert torch.equal(lm_process(x, bias_ids=ids, bias_values=torch.ones(2, 3, device="cuda")), want)
        assert torch.equal(lm_process(x, history=ids, presence_penalty=-1.0), want)
    mask = torch.full((1, 16), -1, dtype=torch.int32, device="cuda")
    got = lm_process(x, mask=mask, mask_rows=torch.tensor([2 ** 32, 0]))
    assert torch.isneginf(got[0]).all() and torch.equal(got[1], x[1])
    got = lm_process(x, history=torch.full((2, 1), 7, dtype=torch.int32, device="cuda"), history_len=torch.tensor([2 ** 32, 2 ** 31]), presence_penalty=-1.0)
    assert torch.equal(got, want)


def lm_process(*args, **kw):
    return logits.process_logits(*args, **kw)
