"""Penalties, biases, grammar masks and the arg-max against a plain implementation in 64 bits.  Tolerance: five steps, each rounded to
32 bits (half a step, 2^-24 of the largest value on the way)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rules64(x, hist, total, prompt, rep, pres, freq, ids, vals, mask, mask_row):
    """(result, largest magnitude on the way); None: the rule is not asked for"""
    x = x.double().cpu()
    b, v = x.shape
    size = x.abs().nan_to_num(0, 0, 0)
    for i in range(b):
        if hist is not None:
            h = [t for t in hist[i, :max(0, total[i])].tolist()]
            p = 0 if prompt is None else min(max(0, int(prompt[i])), len(h))
            count = {}
            for t in h[p:]:
                if 0 <= t < v:
                    count[t] = count.get(t, 0) + 1
            r, a, f = (1.0 if rep is None else float(rep[i]), 0.0 if pres is None else float(pres[i]), 0.0 if freq is None else float(freq[i]))
            for t in {t for t in h if 0 <= t < v}:
                y = float(x[i, t])
                y = y / r if y > 0 else y * r
                steps = [abs(y), abs(y - f * count.get(t, 0)), abs(f * count.get(t, 0))]
                y -= f * count.get(t, 0)
                if t in count:
                    y -= a
                x[i, t] = y
                size[i, t] = max([float(size[i, t]), abs(a), abs(y)] + steps)
        if ids is not None:
            for t, w in {t: w for t, w in zip(ids[i].tolist(), vals[i].tolist()) if 0 <= t < v}.items():
                x[i, t] += w
                size[i, t] = max(float(size[i, t]), abs(w), abs(float(x[i, t])))
        if mask is not None:
            m = i if mask_row is None else int(mask_row[i])
            if 0 <= m < mask.shape[0]:
                w = mask[m].long().cpu() & 0xFFFFFFFF
                bits = ((w[:, None] >> torch.arange(32)) & 1).flatten()[:v]
                x[i][bits == 0] = float("-inf")
    return x, size


def inputs(seed, b, v, length, bias, masks, f32=False, pitch=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(b, v + pitch, generator=g, device=DEV) * 3
    x = (x if f32 else x.bfloat16())[:, :v]
    s = dict(logits=x)
    if length:
        hist = torch.randint(-2, v + 3, (b, length), generator=g, device=DEV).int()
        hist[:, ::3] = hist[:, :1] % v                 # one token over and over
        total = torch.randint(0, length + 3, (b,), generator=g, device=DEV).int()
        s.update(history=hist, n_tokens=total, n_prompt=(total // 2).int(), repetition=1 + torch.rand(b, generator=g, device=DEV),
                 presence=torch.randn(b, generator=g, device=DEV), frequency=torch.randn(b, generator=g, device=DEV))
    if bias:
        s.update(bias_ids=torch.randint(-3, v + 2, (b, bias), generator=g, device=DEV).int(), bias_values=torch.randn(b, bias, generator=g, device=DEV) * 5)
        s["bias_ids"][:, -1] = s["bias_ids"][:, 0]
    if masks:
        s["mask"] = torch.randint(-2**31, 2**31 - 1, (masks, (v + 31) // 32), generator=g, device=DEV).int()
        s["mask_row"] = torch.randint(-1, masks + 1, (b,), generator=g, device=DEV).int()
    return s


def check(s):
    from ixrun_b200.logits import apply_rules

    b, v = s["logits"].shape
    token = torch.full((b,), -9, dtype=torch.int64, device=DEV)
    before = s["logits"].clone()
    out = apply_rules(**s, token=token)
    assert torch.equal(s["logits"], before)
    hist = s.get("history")
    total = None if hist is None else s["n_tokens"].clamp(max=hist.shape[1]).tolist()
    want, size = rules64(s["logits"], None if hist is None else hist.cpu(), total, s.get("n_prompt"), s.get("repetition"), s.get("presence"),
                         s.get("frequency"), s.get("bias_ids"), s.get("bias_values"), s.get("mask"), s.get("mask_row"))
    got = out.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    assert ((got - want).abs()[fine] <= (5 * 2.0 ** -24 * size)[fine]).all()
    # the lowest index of the largest of the results themselves
    top = torch.where(out == out.amax(-1, keepdim=True), torch.arange(v, device=DEV), v).amin(-1)
    assert torch.equal(token, top)
    return out, token


@pytest.mark.parametrize("b,v,length,bias,masks,f32,pitch", [
    (1, 1, 1, 0, 0, True, 0), (1, 7, 5, 3, 1, False, 0), (3, 33, 0, 0, 2, False, 0), (2, 255, 40, 0, 0, True, 1), (5, 4096, 700, 17, 3, False, 8),
    (1, 73448, 1100, 0, 0, False, 0), (17, 8001, 100, 40, 9, True, 0), (4, 151936, 3000, 300, 4, False, 0), (2, 393216, 50, 5, 1, False, 0),
    (1, 262144, 20000, 2047, 1, True, 4), (64, 1000, 64, 1, 64, False, 0), (3, 5000, 0, 9, 0, True, 0), (2, 640, 5, 0, 0, False, 24)])
def test_rules(b, v, length, bias, masks, f32, pitch):
    check(inputs(b * v + length, b, v, length, bias, masks, f32, pitch))


@pytest.mark.parametrize("left", ["repetition", "presence", "frequency", "n_prompt"])
def test_a_penalty_that_is_left_out(left):
    s = inputs(5, 4, 3000, 200, 0, 0)
    s[left] = None
    check(s)


def test_in_place_and_into_wider_rows():
    from ixrun_b200.logits import apply_rules

    s = inputs(6, 3, 1000, 50, 4, 2, f32=True)
    want, token = check(s)
    wide = torch.full((3, 1010), 7.0, device=DEV)
    apply_rules(**s, out=wide[:, 3:1003])
    assert torch.equal(wide[:, 3:1003], want) and (wide[:, :3] == 7).all() and (wide[:, 1003:] == 7).all()
    x = s["logits"]
    t2 = torch.empty_like(token)
    assert apply_rules(**s, out=x, token=t2).data_ptr() == x.data_ptr()
    assert torch.equal(x, want) and torch.equal(t2, token)


def test_ties_infinities_and_rows_without_a_token():
    from ixrun_b200.logits import apply_rules

    v, inf, nan = 5000, float("inf"), float("nan")
    x = torch.zeros(8, v, device=DEV)
    x[0, 4000], x[0, 17], x[0, 4999] = 3.0, 3.0, 3.0
    x[1] = -inf
    x[2, 100], x[2, 2000] = inf, inf
    x[3, 3000], x[3, 70], x[3, 8] = nan, nan, inf
    x[4] = -0.0
    x[4, 9] = 0.0
    x[5] = -inf
    x[5, 4998] = -1e38
    x[6] = 5.0
    x[7] = -1.0
    mask = torch.full((2, (v + 31) // 32), -1, dtype=torch.int32, device=DEV)
    mask[1] = 0
    row = torch.tensor([0, 0, 0, 0, 0, 0, 1, -1], dtype=torch.int32, device=DEV)
    token = torch.empty(8, dtype=torch.int64, device=DEV)
    out = apply_rules(x, mask=mask, mask_row=row, token=token)
    assert token.tolist() == [17, 0, 100, 70, 0, 4998, 0, 0]
    assert (out[6] == -inf).all() and torch.equal(out[:6].nan_to_num(9), x[:6].nan_to_num(9)) and torch.equal(out[7], x[7])


def test_a_graph_takes_what_the_history_has_become():
    from ixrun_b200.logits import apply_rules

    s = inputs(9, 2, 2000, 30, 0, 0)
    out, token = torch.empty(2, 2000, device=DEV), torch.empty(2, dtype=torch.int64, device=DEV)
    s["n_tokens"].fill_(10)
    apply_rules(**s, out=out, token=token)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        apply_rules(**s, out=out, token=token)
    s["n_tokens"].fill_(25)
    graph.replay()
    want, t = check(s)
    assert torch.equal(out, want) and torch.equal(token, t)


@pytest.mark.parametrize("b,v", [(1, 1), (4096, 33), (3, 393216), (2, 31), (300, 5001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_smallest_and_largest_sizes_and_empty_rules(b, v, dtype):
    from ixrun_b200.logits import apply_rules

    x = torch.randn(b, v, generator=torch.Generator(device="cuda").manual_seed(b), device="cuda").to(dtype)
    f, token = x.float(), torch.empty(b, dtype=torch.int64, device="cuda")
    none, zero = torch.empty(b, 0, dtype=torch.int32, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda")
    best = (f == f.max(1, keepdim=True).values).int().argmax(1)                # the lowest index of the largest value
    for rules in ({}, {"history": none, "n_tokens": zero}, {"bias_ids": none, "bias_values": none.float()},
                  {"mask": torch.empty(0, (v + 31) // 32, dtype=torch.int32, device="cuda"), "mask_row": zero - 1}):
        token.fill_(-7)
        assert torch.equal(apply_rules(x, token=token, **rules), f)
        assert torch.equal(token, best)
    # a history that is shorter than its lengths say, with numbers outside the vocabulary
    h = torch.randint(-5, v + 5, (b, 9), dtype=torch.int32, device="cuda")
    got = apply_rules(x, h, zero + 100, zero + 3, presence=torch.ones(b, device="cuda"))
    want = f.clone()
    for i in range(b):
        want[i, sorted({t for t in h[i, 3:].tolist() if 0 <= t < v})] -= 1.0
    assert torch.equal(got, want)


def test_refusals():
    from ixrun_b200 import _lib
    from ixrun_b200.logits import apply_rules

    s = inputs(1, 2, 100, 10, 3, 2)
    for bad in (dict(logits=s["logits"].half()), dict(logits=s["logits"][0]), dict(history=s["history"].long()), dict(n_tokens=None), dict(n_tokens=s["n_tokens"][:1]),
                dict(repetition=s["repetition"].double()), dict(bias_values=None), dict(bias_ids=s["bias_ids"][:, :2]), dict(mask=s["mask"][:, :3]),
                dict(mask=None), dict(mask_row=s["mask_row"].cpu()), dict(out=torch.empty(2, 99, device=DEV)), dict(out=torch.empty(2, 100, device=DEV).bfloat16()),
                dict(token=torch.empty(2, dtype=torch.int32, device=DEV)), dict(logits=s["logits"].t().contiguous().t()),
                dict(history=None)):
        with pytest.raises(ValueError):
            apply_rules(**{**s, **bad})
    with pytest.raises(ValueError):
        apply_rules(s["logits"], mask=s["mask"][:1])
    with pytest.raises(ValueError):
        apply_rules(s["logits"][:0])
    with pytest.raises(_lib.IxbError):
        apply_rules(torch.zeros(1, 400000, device=DEV))


@pytest.mark.parametrize("b,v,length,f32", [(3, 20000, 1537, False), (2, 151936, 9000, True), (5, 65, 3000, False), (1, 300000, 16384, False), (2, 999, 16383, True)])
def test_long_histories(b, v, length, f32):
    """histories that the parts of a row share among themselves, and those that 16 bits do not count"""
    s = inputs(v + length, b, v, length, 7, 0, f32=f32)
    s["history"][:, length // 2:] = v - 1              # one token more often than 13 bits hold, for the longest
    s["n_tokens"].fill_(length)
    s["n_prompt"].fill_(length // 3)
    check(s)


@pytest.mark.parametrize("penalty", ["frequency", "presence"])
@pytest.mark.parametrize("length,v", [(4, 5), (17000, 4096)])
def test_an_infinite_penalty_reaches_generated_tokens_only(penalty, length, v):
    """not those of the prompt, nor those that a bias names; both widths of counters, single logits and eight at a time"""
    from ixrun_b200.logits import apply_rules

    inf = float("inf")
    x = torch.arange(v, dtype=torch.float32, device=DEV)[None] + 1.0
    hist = torch.full((1, length), 1, dtype=torch.int32, device=DEV)           # a token of the prompt, then one that was generated
    hist[0, length // 2:] = 2
    out, token = torch.empty(1, v, device=DEV), torch.empty(1, dtype=torch.int64, device=DEV)
    apply_rules(x, hist, torch.tensor([length], dtype=torch.int32, device=DEV), torch.tensor([length // 2], dtype=torch.int32, device=DEV),
                bias_ids=torch.tensor([[0, 2]], dtype=torch.int32, device=DEV), bias_values=torch.ones(1, 2, device=DEV), out=out, token=token,
                **{penalty: torch.full((1,), inf, device=DEV)})
    want = x.clone()
    want[0, 0], want[0, 2] = 2.0, -inf
    assert torch.equal(out, want) and token.item() == v - 1


def test_dependent_launches_give_the_same_bits():
    """each call in place on the logits of the one before, without a wait of the host"""
    from ixrun_b200.logits import apply_rules
    from ixrun_b200.p6 import set_pdl

    s = [inputs(i, 9, 30000, 500 * i, 40, 3, f32=True) for i in range(1, 5)]
    first = s[0].pop("logits").clone()
    for r in s[1:]:
        r.pop("logits")

    def run(wait):
        x, tokens = first.clone(), []
        for r in s:
            tokens.append(torch.empty(9, dtype=torch.int64, device=DEV))
            wait()
            apply_rules(x, **r, out=x, token=tokens[-1])
        wait()
        return [x] + tokens

    want = run(torch.cuda.synchronize)
    prev = set_pdl(True)
    try:
        for _ in range(10):
            assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))
    finally:
        torch.cuda.synchronize()
        set_pdl(prev)
