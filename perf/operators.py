"""The operators between the projection and the sampler, as cases whose time and results can be measured: the microscaled 4-bit
weight (``quantize_nvfp4`` and its values), the vocabulary projection with such a weight (``lm_head``), and the logits' processing in
front of the sampler (``process_logits``: penalties for repeated tokens, biases, grammar masks).

With ``own`` a case makes the calls a user makes of the framework; without, it is computed in elementary torch operations. Sizes are those of
the benchmark configurations and of the tests: vocabularies of 151,936 / 262,144 / 32,768 (and the odd 20,011 and 4,099), one row to 4096
rows, hidden sizes of 1024 to 4096, histories of up to 2048 tokens.
"""
from __future__ import annotations

import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = 16                               # elements that share a scale
LARGEST = 2688.0                         # the largest e2m1 value times the largest e4m3 scale: 6 * 448


def listed():
    return [
        # A head loaded in BF16 and kept in 4 bits: the whole weight, its scale found on the way.
        dict(name="quantize-151936x4096", kind="quantize", rows=151936, hidden=4096, dtype="bf16", given=False),
        # A small FP32 matrix (a draft model's head) under a scale that came with the checkpoint.
        dict(name="quantize-4099x1024-fp32", kind="quantize", rows=4099, hidden=1024, dtype="fp32", given=True),
        # One stream, a small head: the smallest projection of a decode loop.
        dict(name="head-1-32768x2048", kind="head", rows=1, hidden=2048, vocab=32768, norm=False),
        # The 8 rows of a speculative round, final norm fused.
        dict(name="head-8-151936x4096", kind="head", rows=8, hidden=4096, vocab=151936, norm=True),
        # A few more streams than a tile has rows, over a vocabulary that is no multiple of anything.
        dict(name="head-20-20011x1024", kind="head", rows=20, hidden=1024, vocab=20011, norm=True),
        # A serving batch.
        dict(name="head-256-151936x4096", kind="head", rows=256, hidden=4096, vocab=151936, norm=False),
        # One stream: FP32 logits, penalties over the tokens so far.
        dict(name="logits-1-fp32", kind="logits", rows=1, vocab=151936, dtype="fp32", hist=2048, shared=False, bias=0, mask="none", place="new"),
        # The 8 rows of a speculative round under a grammar: one history that grows by a draft from row to row, a mask to each row.
        dict(name="logits-8-round", kind="logits", rows=8, vocab=151936, dtype="bf16", hist=2048, shared=True, bias=0, mask="grammar", place="new"),
        # Odd sizes: rows at odd addresses, short and empty histories, a row whose mask leaves nothing.
        dict(name="logits-37-odd-fp32", kind="logits", rows=37, vocab=20011, dtype="fp32", hist=257, shared=False, bias=33, mask="mixed", place="new"),
        # Requests under grammars only, in place (most of the vocabulary is masked): the large-vocabulary configuration.
        dict(name="mask-64-262144", kind="logits", rows=64, vocab=262144, dtype="bf16", hist=0, shared=False, bias=0, mask="grammar", place="same"),
        # The batched configuration with everything on: penalties by request, biases of up to 300 tokens, some rows under a grammar.
        dict(name="logits-256-all", kind="logits", rows=256, vocab=151936, dtype="bf16", hist=2048, shared=False, bias=300, mask="mixed", place="new"),
        # The large batch that the benchmark is quoted on.
        dict(name="logits-4096", kind="logits", rows=4096, vocab=151936, dtype="bf16", hist=2048, shared=False, bias=0, mask="none", place="new"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("quantize", "head", "head", "logits", "logits"))
    if kind == "quantize":
        return dict(kind=kind, rows=_log_int(rng, 64, 131072), hidden=16 * _log_int(rng, 4, 256), dtype=rng.choice(("bf16", "bf16", "fp32")), given=rng.random() < 0.5)
    if kind == "head":
        return dict(kind=kind, rows=_log_int(rng, 1, 256), hidden=64 * _log_int(rng, 4, 64), vocab=_log_int(rng, 4000, 151936), norm=rng.random() < 0.5)
    rows, vocab = _log_int(rng, 1, 2048), _log_int(rng, 4000, 262144)
    place = rng.choice(("new", "new", "new", "same"))
    hist = 0 if place == "same" else rng.choice((0, _log_int(rng, 1, 4096), _log_int(rng, 64, 4096)))
    bias = 0 if place == "same" else rng.choice((0, 0, _log_int(rng, 1, 300)))
    mask = "grammar" if place == "same" or (hist == 0 and bias == 0) else rng.choice(("none", "grammar", "mixed"))
    return dict(kind="logits", rows=rows, vocab=vocab if rng.random() < 0.5 else (vocab + 63) // 64 * 64, dtype=rng.choice(("bf16", "bf16", "fp32")), hist=hist,
                shared=hist > 16 and rows <= 16 and rng.random() < 0.5, bias=bias, mask=mask, place=place)


def _dtype(case):
    return torch.bfloat16 if case.get("dtype", "bf16") == "bf16" else torch.float32


# ---- the 4-bit format in elementary operations (64 bits: a value next to a border between two codes must fall on its own side) ----------

def _round_e4m3(t):
    """Nearest e4m3 value, ties to even, of doubles >= 0; saturates at 448."""
    _, e = torch.frexp(t)                                       # t = m 2^e, m in [0.5, 1)
    step = torch.ldexp(torch.ones_like(t), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(t / step) * step, max=448.0)


def _magnitude_code(q):
    """Code of the nearest e2m1 magnitude, ties to the even code."""
    return ((q > 0.25).to(torch.uint8) + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5) + (q > 5.0)).to(torch.uint8)


def _global_scale(x):
    a = x.abs().amax().double()
    g = (a / torch.full_like(a, LARGEST)).float()
    return torch.where(g >= 2.0 ** -126, g, torch.ones_like(g)).reshape(1)


def _quantize(x, g):
    """Codes [rows, H] (sign in bit 3) and e4m3 scales [rows, H / 16] as doubles, in pieces of rows."""
    rows, H = x.shape
    codes = torch.empty(rows, H, dtype=torch.uint8, device=x.device)
    scales = torch.empty(rows, H // BLOCK, dtype=torch.float64, device=x.device)
    gd = g.double()
    step = max(1, (1 << 26) // H)
    for r in range(0, rows, step):
        b = x[r:r + step].double().reshape(-1, H // BLOCK, BLOCK)
        s = _round_e4m3(b.abs().amax(-1) / (6.0 * gd))
        unit = (s * gd).unsqueeze(-1)
        q = torch.where(unit > 0, b.abs() / unit, torch.zeros_like(b))
        codes[r:r + step] = (_magnitude_code(q) + 8 * (b < 0)).reshape(-1, H).to(torch.uint8)
        scales[r:r + step] = s
    return codes, scales


def _values(codes, scales, g):
    """float32 values of codes and scales."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    rows, H = codes.shape
    out = torch.empty(rows, H, dtype=torch.float32, device=codes.device)
    step = max(1, (1 << 27) // H)
    for r in range(0, rows, step):
        v = table[codes[r:r + step].int()].reshape(-1, H // BLOCK, BLOCK) * scales[r:r + step].float().unsqueeze(-1)
        out[r:r + step] = (v * g).reshape(-1, H)
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)
    kind = case["kind"]
    st = dict(case=case)
    if kind == "quantize":
        x = torch.empty(case["rows"], case["hidden"], dtype=_dtype(case), device=dev)
        step = max(1, (1 << 27) // case["hidden"])
        spread = torch.exp(0.3 * normal(case["rows"], 1)) * 0.05            # rows of a head differ in size
        for r in range(0, case["rows"], step):
            n = min(step, case["rows"] - r)
            x[r:r + n] = (normal(n, case["hidden"]) * spread[r:r + n]).to(x.dtype)
        st["x"] = x
        st["scale"] = _global_scale(x) * 1.25 if case["given"] else None
    elif kind == "head":
        V, H = case["vocab"], case["hidden"]
        codes = torch.empty(V, H // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(V, H // BLOCK, dtype=torch.float8_e4m3fn, device=dev)
        g = torch.full((1,), 0.05 * 5.5 / LARGEST, device=dev) * (1.0 + 0.1 * torch.rand(1, generator=gen, device=dev))
        step = max(1, (1 << 26) // H)
        for r in range(0, V, step):
            n = min(step, V - r)
            c, s = _quantize((normal(n, H) * 0.05), g)
            codes[r:r + n] = c[:, 0::2] | (c[:, 1::2] << 4)
            scales[r:r + n] = s.float().to(torch.float8_e4m3fn)
        st["hidden"] = normal(case["rows"], H).to(torch.bfloat16)
        st["norm"] = (0.1 * normal(H)).to(torch.bfloat16) if case["norm"] else None
        st["codes"], st["scales"], st["scale"] = codes, scales, g
        if own:
            import lithos_metal_b200 as lm
            st["weight"] = lm.Nvfp4Weight(codes, scales, g)
    else:
        rows, V, n = case["rows"], case["vocab"], case["hist"]
        logits = torch.empty(rows, V, dtype=_dtype(case), device=dev)
        step = max(1, (1 << 27) // V)
        for r in range(0, rows, step):
            k = min(step, rows - r)
            logits[r:r + k] = (2.0 * normal(k, V)).to(logits.dtype)
        st["logits"] = logits
        st["out"] = logits if case["place"] == "same" else torch.empty_like(logits)
        uniform = lambda *shape: torch.rand(*shape, generator=gen, device=dev)
        st.update(history=None, history_len=None, prompt_len=None, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None, bias_values=None, mask=None, mask_rows=None)
        if n:
            one = 1 if case["shared"] else rows
            h = (uniform(one, n) ** 3 * V).to(torch.int32).clamp_(max=V - 1)             # some tokens come often
            if case["shared"]:                                                            # row r: the tokens so far and r drafts
                st["history"] = h.expand(rows, n)
                st["history_len"] = torch.arange(n - rows + 1, n + 1, dtype=torch.int32, device=dev)
                st["prompt_len"] = torch.full((rows,), n // 2, dtype=torch.int32, device=dev)
            else:
                length = (uniform(rows) * 1.25 * n).to(torch.int32).clamp_(max=n)
                st["history"], st["history_len"] = h, length
                st["prompt_len"] = (length.float() * uniform(rows)).to(torch.int32)
            per_row = lambda lo, hi: lo + (hi - lo) * uniform(rows)
            st["repetition"], st["presence"], st["frequency"] = per_row(1.0, 1.3), per_row(0.0, 1.0), per_row(0.0, 0.5)
        if case["bias"]:
            ids = torch.randint(0, V, (rows, case["bias"]), generator=gen, device=dev, dtype=torch.int32)
            st["bias_ids"] = torch.where(uniform(rows, case["bias"]) < 0.2, torch.full_like(ids, -1), ids)      # lists of different lengths, padded with -1
            st["bias_values"] = 10.0 * (2.0 * uniform(rows, case["bias"]) - 1.0)
        if case["mask"] != "none":
            words, states = (V + 31) // 32, rows if case["mask"] == "grammar" else max(1, rows // 2)
            bits = torch.empty(states, words, dtype=torch.int32, device=dev)
            shift = torch.arange(32, device=dev)
            step = max(1, (1 << 26) // V)
            for r in range(0, states, step):
                k = min(step, states - r)
                runs = torch.repeat_interleave(uniform(k, (words + 3) // 4) < 0.08, 4, dim=1)[:, :words]     # a grammar's tokens come in runs, and singly
                allowed = (uniform(k, words, 32) < 0.02) | (runs.unsqueeze(-1) & (uniform(k, words, 32) < 0.7))
                bits[r:r + k] = (allowed.long() << shift).sum(-1).to(torch.int32)
            if case["mask"] == "mixed":
                bits[0] = 0                                                               # a state that allows nothing
                st["mask_rows"] = torch.randint(-1, states, (rows,), generator=gen, device=dev, dtype=torch.int32)   # -1: no grammar on the row
                st["mask_rows"][0] = 0
            st["mask"] = bits
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------------------------------

def _run_own(st):
    import lithos_metal_b200 as lm
    kind = st["case"]["kind"]
    if kind == "quantize":
        w = lm.quantize_nvfp4(st["x"], scale=st["scale"])
        return w.dequantize(), w.scale
    if kind == "head":
        return lm.lm_head(st["hidden"], st["weight"], st["norm"])
    return lm.process_logits(st["logits"], history=st["history"], history_len=st["history_len"], prompt_len=st["prompt_len"], repetition_penalty=st["repetition"],
                             presence_penalty=st["presence"], frequency_penalty=st["frequency"], bias_ids=st["bias_ids"], bias_values=st["bias_values"],
                             mask=st["mask"], mask_rows=st["mask_rows"], out=st["out"])


def _counts(ids, keep, vocab):
    """Occurrences of every token among the kept ids of each row."""
    c = torch.zeros(ids.shape[0], vocab, dtype=torch.float32, device=ids.device)
    return c.scatter_add_(1, ids.long(), keep.float())


def run(st):
    if own:
        return _run_own(st)
    kind = st["case"]["kind"]
    if kind == "quantize":
        g = st["scale"] if st["scale"] is not None else _global_scale(st["x"])
        codes, scales = _quantize(st["x"], g)
        return _values(codes, scales, g), g
    if kind == "head":
        x = st["hidden"].float()
        if st["norm"] is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1.0 + st["norm"].float())
            x = x.to(torch.bfloat16).float()                    # (the norm's output is a BF16 tensor by definition)
        c = st["codes"]
        codes = torch.stack((c & 15, c >> 4), dim=-1).reshape(c.shape[0], -1)
        return (x @ _values(codes, st["scales"], st["scale"]).T).to(torch.bfloat16)
    z = st["logits"].float()
    rows, V = z.shape
    if st["history"] is not None:
        at = torch.arange(st["history"].shape[1], device=z.device)
        seen = at < st["history_len"].unsqueeze(1)
        c_all = _counts(st["history"], seen, V)
        c_out = _counts(st["history"], seen & (at >= st["prompt_len"].unsqueeze(1)), V)
        rho, pi, phi = (st[k].unsqueeze(1) for k in ("repetition", "presence", "frequency"))
        z = torch.where(c_all > 0, torch.where(z > 0, z / rho, z * rho), z)
        z = torch.where(c_out > 0, z - pi - phi * c_out, z)
    if st["bias_ids"] is not None:
        ids, on = st["bias_ids"], st["bias_ids"] >= 0
        z = z.scatter_add(1, ids.clamp(min=0).long(), torch.where(on, st["bias_values"], torch.zeros_like(st["bias_values"])))
    if st["mask"] is not None:
        v = torch.arange(V, device=z.device)
        words = st["mask"] if st["mask_rows"] is None else st["mask"][st["mask_rows"].clamp(min=0).long()]
        allowed = (words[:, v >> 5] >> (v & 31)) & 1
        if st["mask_rows"] is not None:
            allowed = allowed | (st["mask_rows"] < 0).int().unsqueeze(1)
        z = torch.where(allowed == 1, z, torch.full_like(z, -math.inf))
    return st["out"].copy_(z)


def work(case):
    kind = case["kind"]
    if kind == "quantize":                                      # read x; write codes, scales and the values they stand for
        n = case["rows"] * case["hidden"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * size + n // 2 + n // BLOCK + 4 * n, "flops": 4 * n}
    if kind == "head":
        n = case["vocab"] * case["hidden"]
        return {"bytes": n // 2 + n // BLOCK + 2 * case["rows"] * (case["hidden"] + case["vocab"]), "flops": 2 * case["rows"] * n}
    rows, V = case["rows"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    lists = (1 if case["shared"] else rows) * 4 * case["hist"] + rows * 8 * case["bias"]
    words = (V + 31) // 32 * 4 * {"none": 0, "grammar": rows, "mixed": max(1, rows // 2)}[case["mask"]]
    logits = rows * V * size * (1 if case["place"] == "same" else 2)       # (in place under a mask: masked logits are written, not read)
    return {"bytes": logits + lists + words, "flops": rows * V}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x = st["x"]
        dev = x.device
        amax = x.abs().max().double().item()
        if st["scale"] is not None:
            g = st["scale"].double().item()
        else:
            g = torch.tensor(amax / LARGEST, dtype=torch.float64).float().double().item()
        e4m3 = torch.arange(127, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn).double()           # the positive values, in order
        e2m1 = torch.tensor(E2M1, dtype=torch.float64, device=dev)

        def nearest(v, grid):                                   # index of the nearest grid value, ties to the even index
            hi = torch.searchsorted(grid, v).clamp(1, len(grid) - 1)
            lo = hi - 1
            below, above = v - grid[lo], grid[hi] - v
            return torch.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)

        out = torch.empty(x.shape, dtype=torch.float64, device=dev)
        step = max(1, (1 << 25) // x.shape[1])
        for r in range(0, x.shape[0], step):
            b = x[r:r + step].double().unflatten(1, (-1, BLOCK))
            s = e4m3[nearest(b.abs().max(-1).values / 6.0 / g, e4m3)].unsqueeze(-1)
            q = torch.where(s > 0, b.abs() / (s * g), torch.zeros_like(b))
            out[r:r + step] = (torch.sign(b) * e2m1[nearest(q, e2m1)] * s * g).flatten(1)
        return out, torch.tensor([g], dtype=torch.float64, device=dev)
    if kind == "head":
        x = st["hidden"].double()
        if st["norm"] is not None:
            x = x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-6) * (1.0 + st["norm"].double())
            x = x.to(torch.bfloat16).double()
        grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
        parts = []
        step = max(1, (1 << 26) // case["hidden"])
        for v in range(0, case["vocab"], step):
            c = st["codes"][v:v + step].long()
            nibbles = torch.empty(c.shape[0], 2 * c.shape[1], dtype=torch.long, device=x.device)
            nibbles[:, 0::2], nibbles[:, 1::2] = c % 16, c // 16
            w = grid[nibbles % 8] * (1 - 2 * (nibbles // 8))
            w = w * st["scales"][v:v + step].double().repeat_interleave(BLOCK, dim=1)
            parts.append(torch.matmul(x, w.T) * st["scale"].double())
        return torch.cat(parts, dim=1)
    logits = st["logits"]
    rows, V = logits.shape
    out = logits.double()
    for r in range(rows):
        z = out[r]
        if st["history"] is not None:
            n, p = int(st["history_len"][r]), int(st["prompt_len"][r])
            ids = st["history"][r, :n].long()
            every, behind = torch.bincount(ids, minlength=V), torch.bincount(ids[p:], minlength=V).double()
            rho, pi, phi = (st[k][r].double() for k in ("repetition", "presence", "frequency"))
            z = torch.where(every > 0, z * torch.where(z > 0, 1.0 / rho, rho), z)
            z = z - torch.where(behind > 0, pi + phi * behind, torch.zeros_like(z))
        if st["bias_ids"] is not None:
            on = st["bias_ids"][r] >= 0
            z = z + torch.bincount(st["bias_ids"][r][on].long(), weights=st["bias_values"][r][on].double(), minlength=V)
        if st["mask"] is not None:
            m = r if st["mask_rows"] is None else int(st["mask_rows"][r])
            if m >= 0:
                word = st["mask"][m].long() & 0xFFFFFFFF
                bits = (word.unsqueeze(1) >> torch.arange(32, device=z.device)).remainder(2).flatten()[:V]
                z = z.masked_fill(bits == 0, -math.inf)
        out[r] = z
    return out
