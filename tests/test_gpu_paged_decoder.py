"""Requests that come and go on a packed model over a paged cache: tables, rotary embedding into pages, paged attention and the
rules on logits together, against the same model with one static cache per sequence.  The two differ in the order of sums and
in the roundings of the attention's probabilities, so logits agree to bf16 noise (the bound that the other decoders' tests take)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def tiny(head_dim=64, max_seq=96):
    from ixrun_b200.llama_runner import LlamaConfig, PackedLlama, synthetic_llama

    cfg = LlamaConfig(n_layers=2, hidden=256, intermediate=512, n_heads=4, n_kv_heads=2, head_dim=head_dim, vocab=1000, max_seq=max_seq)
    return cfg, PackedLlama(cfg, *synthetic_llama(cfg, seed=1), weights="packed")


def prompts_of(cfg, lengths, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab, (n,), generator=g) for n in lengths]


def near(got, ref):
    assert (got - ref).abs().max() <= 0.05 * ref.abs().max()


def near_best(token, ref):
    """With logits off by at most b = 0.05 max |ref|, got[token] >= got[best] says ref[token] + b >= ref[best] - b: the arg-max of
    the one has a logit within 2 b of the other's largest."""
    assert ref.max() - ref.reshape(-1)[token] <= 2 * 0.05 * ref.abs().max()


def check_alone(model, tokens, n_prompt, logits):
    """logits[i]: behind tokens[:n_prompt + i], as the model alone has them"""
    near(logits[0], model.prefill(tokens[:n_prompt])[0])
    for i, got in enumerate(logits[1:]):
        near(got, model.step(tokens[n_prompt + i].cuda(), n_prompt + i)[0])


@pytest.mark.parametrize("requests,head_dim,page", [(3, 64, 16), (3, 128, 64), (12, 64, 32)])
@pytest.mark.parametrize("captured", [False, True])
def test_requests_of_different_lengths_have_the_logits_that_they_have_alone(requests, head_dim, page, captured):
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny(head_dim)
    dec = PagedDecoder(model, requests, requests * (-(-cfg.max_seq // page)), page=page)
    if captured:
        dec.capture()
    prompts = prompts_of(cfg, [1 + 7 * i % 60 for i in range(requests)])
    numbers = [dec.add(p) for p in prompts]
    tokens, logits = {r: p.tolist() for r, p in zip(numbers, prompts)}, {r: [] for r in numbers}
    for _ in range(5):
        new = dec.step().tolist()
        assert min(new) >= 0
        for r in numbers:
            logits[r].append(dec.logits[r].clone())
            assert int(logits[r][-1].argmax()) == new[r]
            tokens[r].append(new[r])
    assert dec.pages.length.tolist() == [p.numel() + 4 for p in prompts] == dec._cached
    for r, p in list(zip(numbers, prompts))[:4]:
        check_alone(model, torch.tensor(tokens[r]), p.numel(), logits[r])


def run_of_requests(dec, prompts, max_rows):
    """(numbers, tokens and logits of every step): two requests, a third while they answer, the first goes, a fourth takes its place"""
    out = []

    def steps(n):
        for _ in range(n):
            tok = dec.step(max_rows)
            out.append((tok.clone(), torch.where((tok >= 0)[:, None], dec.logits, 0.0)))

    numbers = [dec.add(prompts[0]), dec.add(prompts[1])]
    steps(6)
    numbers.append(dec.add(prompts[2]))
    steps(6)
    dec.remove(numbers[0])
    numbers.append(dec.add(prompts[3]))
    steps(6)
    return numbers, out


@pytest.mark.parametrize("max_rows", [2048, 7])
def test_requests_that_come_and_go(max_rows):
    """Prompts in one pass and in pieces of a few rows beside the answers of others; a number that is taken again; eager and captured:
    the same bits."""
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny()
    prompts = prompts_of(cfg, (17, 5, 30, 9))
    dec = PagedDecoder(model, 3, 10, page=16)
    numbers, out = run_of_requests(dec, prompts, max_rows)
    assert numbers == [0, 1, 2, 0]
    fast = PagedDecoder(model, 3, 10, page=16).capture()
    n2, out2 = run_of_requests(fast, prompts, max_rows)
    assert n2 == numbers
    for a, b in zip(out, out2):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert dec.pages.n_free.item() == dec._pages_left and dec.pages.length.tolist() == dec._cached
    for i, (r, first, last) in enumerate([(0, 0, 12), (1, 0, 18), (2, 6, 18), (0, 12, 18)]):
        mine = [(int(t[r]), lg[r]) for t, lg in out[first:last] if int(t[r]) >= 0]
        fed = -(-prompts[i].numel() // max_rows)
        assert last - first - fed - 4 <= len(mine) <= last - first             # (others' pieces come before a later number's)
        check_alone(model, torch.cat([prompts[i], torch.tensor([t for t, _ in mine])]), prompts[i].numel(), [lg for _, lg in mine])
    for r in range(3):
        dec.remove(r)
    assert dec.pages.n_free.item() == 10 == dec._pages_left
    assert sorted(dec.pages.free.tolist()) == list(range(10))


def test_rules_of_a_request_are_its_own():
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny()
    p = prompts_of(cfg, (20,))[0]
    dec = PagedDecoder(model, 5, 20, page=32, max_bias=3)
    allowed = torch.zeros(cfg.vocab, dtype=torch.bool)
    allowed[[3, 31, 32, 999]] = True
    plain, grammar, biased, never_twice = dec.add(p), dec.add(p, allowed=allowed), dec.add(p, bias={7: 1e4, 8: 9e3}), dec.add(p, presence=1e4)
    seen = {r: [] for r in (plain, grammar, biased, never_twice)}
    for i in range(12):
        if i == 6:
            dec.allow(grammar, torch.arange(cfg.vocab) == 500)
        if i == 9:
            dec.allow(grammar, None)
        for r, t in enumerate(dec.step().tolist()):
            if r in seen:
                seen[r].append(t)
            else:
                assert t == -1
    assert set(seen[grammar][:6]) <= {3, 31, 32, 999} and seen[grammar][6:9] == [500] * 3 and seen[grammar][9] != 500
    assert seen[biased] == [7] * 12
    assert len(set(seen[never_twice])) == 12
    assert seen[plain][0] == seen[never_twice][0]
    near_best(seen[plain][0], model.prefill(p))
    # the next request of a number has none of its predecessor's rules
    dec.remove(biased)
    assert dec.add(p) == biased
    assert int(dec.step()[biased]) == seen[plain][0]


def test_generate_with_more_prompts_than_numbers_and_pages():
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny()
    prompts = prompts_of(cfg, (40, 3, 18, 90, 1, 25, 96))
    dec = PagedDecoder(model, 2, 7, page=16).capture()
    out = dec.generate(prompts, 10)
    assert [len(o) for o in out] == [10, 10, 10, 7, 10, 10, 1]                # (of 96 tokens there is room for all but the last one's own)
    assert dec.pages.n_free.item() == 7 and dec.generate(prompts, 10) == out
    for p, o in zip(prompts, out):
        near_best(o[0], model.prefill(p))
    eos = out[0][4]
    assert dec.generate(prompts[:1], 10, eos=eos) == [out[0][:out[0].index(eos) + 1]]
    assert dec.generate([], 3) == []


def test_refusals():
    from ixrun_b200.llama_runner import PackedLlama, PagedDecoder, synthetic_llama

    cfg, model = tiny()
    with pytest.raises(ValueError):
        PagedDecoder(PackedLlama(cfg, *synthetic_llama(cfg, seed=1), weights="decoded"), 2, 4)
    for bad in (dict(requests=0), dict(requests=65), dict(n_pages=0), dict(page=48), dict(max_bias=-1)):
        with pytest.raises(ValueError):
            PagedDecoder(model, **{**dict(requests=2, n_pages=4, page=16), **bad})
    dec = PagedDecoder(model, 2, 4, page=16)
    ids = torch.arange(20)
    with pytest.raises(RuntimeError, match="no request"):
        dec.step()
    for bad in (dict(prompt=ids[:0]), dict(prompt=torch.zeros(97, dtype=torch.long)), dict(prompt=ids.float()), dict(prompt=torch.tensor([5, -1])),
                dict(prompt=torch.tensor([cfg.vocab])), dict(repetition=0.0), dict(bias={i: 1.0 for i in range(65)}), dict(allowed=torch.ones(5, dtype=torch.bool))):
        with pytest.raises(ValueError):
            dec.add(**{"prompt": ids, **bad})
    assert dec._known == [None, None]
    with pytest.raises(ValueError):
        dec.remove(0)
    a, b = dec.add(ids), dec.add(torch.arange(40))
    with pytest.raises(RuntimeError, match="taken"):
        dec.add(ids)
    with pytest.raises(RuntimeError, match="5 pages, 4 are left"):
        dec.step()
    with pytest.raises(RuntimeError, match="itself"):
        dec.generate([ids], 2)
    assert dec.pages.n_free.item() == 4 and dec._cached == [0, 0]
    dec.remove(b)
    first = dec.step()[a].item()
    near_best(first, model.prefill(ids))
    # a request with all the tokens that fit
    dec = PagedDecoder(model, 2, 6, page=16)
    full = dec.add(torch.arange(96))
    assert dec.step()[full] >= 0
    with pytest.raises(RuntimeError, match="96 tokens"):
        dec.step()
    dec.capture()
    dec.remove(full)
    dec.add(ids)
    assert dec.step()[0].item() == first
    assert dec.step()[0].item() >= 0


def test_a_step_of_no_rows_is_refused_and_changes_nothing():
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny()
    dec = PagedDecoder(model, 2, 8, page=16)
    r = dec.add(torch.arange(5))
    for rows in (0, -1, -7):
        with pytest.raises(ValueError):
            dec.step(rows)
    assert dec._cached == [0, 0] == dec.pages.length.tolist() and dec._known == [5, None] and dec._pages_left == 8
    dec.remove(r)
    with pytest.raises(ValueError):
        dec.generate([torch.arange(5)], 2, max_rows=0)
    assert dec._known == [None, None]


@pytest.mark.parametrize("rows", [1, 3, 4])
def test_every_request_gets_on_where_there_are_fewer_rows_than_requests(rows):
    """answers and prompts in turns, with the logits that each has alone"""
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny()
    dec = PagedDecoder(model, 8, 48, page=16).capture()
    prompts = prompts_of(cfg, (3, 1, 1, 9, 1, 1, 1, 2))
    tokens, logits = [p.tolist() for p in prompts], [[] for _ in prompts]
    for p in prompts:
        dec.add(p)
    for _ in range(60):
        for r, t in enumerate(dec.step(rows).tolist()):
            if t >= 0:
                tokens[r].append(t)
                logits[r].append(dec.logits[r].clone())
    assert min(len(x) for x in logits) >= 2
    for r in (0, 3, 7):
        check_alone(model, torch.tensor(tokens[r]), prompts[r].numel(), logits[r])


def test_rules_that_leave_no_token_are_refused():
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny()
    inf, ids = float("inf"), torch.arange(9)
    one = torch.zeros(cfg.vocab, dtype=torch.bool)
    none = one.clone()
    one[7] = True
    dec = PagedDecoder(model, 2, 8, page=16, max_bias=4)
    for bad in (dict(allowed=none), dict(allowed=none.cuda()), dict(allowed=one, bias={7: -inf}), dict(allowed=one, bias={7: -1e39, 3: 1.0}),
                dict(bias={5: float("nan")}), dict(presence=inf), dict(frequency=float("nan")), dict(repetition=inf), dict(repetition=1e-60)):
        with pytest.raises(ValueError):
            dec.add(ids, **bad)
    assert dec._known == [None, None] and dec.mask_row.tolist() == [-1, -1]
    r, b = dec.add(ids, allowed=one, bias={8: -inf, -1: -inf}), dec.add(ids, bias={3: -inf})
    assert dec.step()[r] == 7
    for mask in (none, torch.arange(cfg.vocab) == 8):
        with pytest.raises(ValueError):
            dec.allow(r, mask)
    assert dec.step()[r] == 7                          # (the mask that it had)
    dec.allow(b, torch.arange(cfg.vocab) == 8)         # (another request's ban)
    assert dec.step().tolist() == [7, 8]
    # the next request of the number is not bound by its predecessor's bans
    dec.remove(r)
    assert dec.add(ids, allowed=torch.arange(cfg.vocab) == 8) == r
    assert dec.step()[r] == 8


@pytest.mark.parametrize("last", ["token", "length", "empty", "rules"])
def test_generate_that_refuses_a_prompt_leaves_no_request_behind(last):
    from ixrun_b200.llama_runner import PagedDecoder

    cfg, model = tiny()
    dec = PagedDecoder(model, 2, 12, page=16)
    ids = torch.arange(5)
    bad = {"token": torch.tensor([cfg.vocab]), "length": torch.zeros(cfg.max_seq + 1, dtype=torch.long), "empty": ids[:0], "rules": ids}[last]
    with pytest.raises(ValueError):
        dec.generate([ids, ids, ids, bad], 3, **({"bias": {i: 0.5 for i in range(65)}} if last == "rules" else {}))
    assert dec._known == [None, None] and dec._pages_left == 12 == dec.pages.n_free.item()
    assert [len(o) for o in dec.generate([ids, ids, ids], 3)] == [3, 3, 3]


@pytest.mark.parametrize("captured", [False, True])
def test_dependent_launches_give_the_same_bits(captured):
    from ixrun_b200.llama_runner import PagedDecoder
    from ixrun_b200.p6 import set_pdl

    cfg, model = tiny()
    prompts = prompts_of(cfg, (17, 5, 30, 9))
    numbers, want = run_of_requests(PagedDecoder(model, 3, 10, page=16), prompts, 7)
    prev = set_pdl(True)
    try:
        dec = PagedDecoder(model, 3, 10, page=16)
        n2, got = run_of_requests(dec.capture() if captured else dec, prompts, 7)
    finally:
        torch.cuda.synchronize()
        set_pdl(prev)
    assert n2 == numbers
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
