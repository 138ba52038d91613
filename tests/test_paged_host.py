"""Argument checks of the paged-cache and logits entry points, on the CPU: they come before any CUDA call."""
import ctypes

import pytest
import torch

P = 4096                                               # a pointer that no call gets as far as to use


def call(name, **changed):
    from ixrun_b200 import _lib

    args = dict(ARGS[name])
    assert set(changed) <= set(args), changed
    args.update(changed)
    rc = getattr(_lib.lib(), name)(*args.values())
    return rc, _lib.lib().ixb_last_error().decode()


ARGS = {
    "ixb_page_step": dict(q_len=P, length=P, table=P, free=P, n_free=P, requests=2, width=3, n_pages=4, page=16, rows=5, cu_rows=P, new_length=P,
                          new_n_free=P, slot=P, pos=P, owner=P, status=P, stream=None),
    "ixb_page_release": dict(done=P, length=P, table=P, free=P, n_free=P, requests=2, width=3, n_pages=4, page=16, status=P, stream=None),
    "ixb_rope_paged": dict(q=P, k=P, v=P, pos=P, slot=P, k_pages=P, v_pages=P, q_norm=None, k_norm=None, cos=P, sin=P, out=P, rows=3, hq=4, hkv=2,
                           head_dim=64, rot_dim=64, eps=1e-6, q_stride=256, kv_stride=128, out_stride=256, max_seq=9, n_pages=4, page=16,
                           k_page_stride=2048, v_page_stride=2048, stream=None),
    "ixb_attn_paged": dict(q=P, k_pages=P, v_pages=P, table=P, length=P, cu_rows=P, out=P, requests=2, width=3, rows=5, max_q=5, hq=4, hkv=2, head_dim=64,
                           n_pages=4, page=16, q_stride=256, k_page_stride=2048, v_page_stride=2048, scale=0.1, scratch=P, scratch_bytes=1 << 40,
                           stream=None),
    "ixb_logits": dict(logits=P, f32=0, pitch=64, history=P, hist_len=7, hist_pitch=7, n_tokens=P, n_prompt=P, repetition=None, presence=None, frequency=None,
                       bias_ids=None, bias_values=None, n_bias=0, mask=None, n_masks=0, mask_pitch=0, mask_row=None, out=P, out_pitch=64, token=P, rows=1,
                       vocab=64, stream=None),
}
BAD = [
    ("ixb_page_step", dict(q_len=None), 1), ("ixb_page_step", dict(status=None), 1), ("ixb_page_step", dict(requests=0), 2),
    ("ixb_page_step", dict(requests=4097), 2), ("ixb_page_step", dict(page=24), 2), ("ixb_page_step", dict(page=512), 2), ("ixb_page_step", dict(rows=-1), 1),
    ("ixb_page_step", dict(slot=None), 1), ("ixb_page_step", dict(n_pages=1 << 28), 1), ("ixb_page_step", dict(width=0), 1),
    ("ixb_page_release", dict(done=None), 1), ("ixb_page_release", dict(page=0), 2), ("ixb_page_release", dict(n_pages=0), 1),
    ("ixb_rope_paged", dict(slot=None), 1), ("ixb_rope_paged", dict(head_dim=96), 2), ("ixb_rope_paged", dict(rot_dim=66), 1),
    ("ixb_rope_paged", dict(rot_dim=33), 1), ("ixb_rope_paged", dict(q_stride=255), 1), ("ixb_rope_paged", dict(kv_stride=64), 1),
    ("ixb_rope_paged", dict(v_page_stride=2040), 1), ("ixb_rope_paged", dict(rows=0), 1), ("ixb_rope_paged", dict(page=17), 2),
    ("ixb_attn_paged", dict(scratch=None), 1), ("ixb_attn_paged", dict(hq=5), 1), ("ixb_attn_paged", dict(head_dim=80), 2), ("ixb_attn_paged", dict(rows=0), 1),
    ("ixb_attn_paged", dict(max_q=0), 1), ("ixb_attn_paged", dict(q_stride=260), 1), ("ixb_attn_paged", dict(k_page_stride=2052), 1),
    ("ixb_attn_paged", dict(q=P + 8), 1), ("ixb_attn_paged", dict(out=P + 2), 1), ("ixb_attn_paged", dict(scratch_bytes=4096), 4),
    ("ixb_attn_paged", dict(requests=5000), 2),
    ("ixb_logits", dict(logits=None), 1), ("ixb_logits", dict(n_tokens=None), 1), ("ixb_logits", dict(pitch=63), 1), ("ixb_logits", dict(out_pitch=63), 1),
    ("ixb_logits", dict(vocab=393217, pitch=400000, out_pitch=400000), 2), ("ixb_logits", dict(hist_pitch=6), 1), ("ixb_logits", dict(n_bias=3), 1),
    ("ixb_logits", dict(n_bias=2048, bias_ids=P, bias_values=P), 2), ("ixb_logits", dict(mask=P, n_masks=1, mask_pitch=1), 1),
    ("ixb_logits", dict(hist_len=1 << 20, hist_pitch=1 << 20), 2), ("ixb_logits", dict(rows=0), 1),
]


@pytest.mark.parametrize("name,changed,code", BAD, ids=lambda v: str(v) if not isinstance(v, dict) else "-".join(v))
def test_bad_arguments_are_refused_before_any_cuda_call(name, changed, code):
    rc, text = call(name, **changed)
    assert rc == code and text


@pytest.mark.parametrize("requests,rows,hq,page,width,fits", [
    (4096, 4096, 4, 256, 1 << 22, False),              # 4096 requests that share a table's pages, 2^30 positions each
    (64, 2048, 16, 256, 1 << 22, False), (4096, 4096, 16, 16, 1 << 15, True), (1, 1, 16, 256, (1 << 23) - 1, True), (64, 16384, 16, 64, 1 << 14, True)])
def test_work_that_32_bits_do_not_count_is_refused(requests, rows, hq, page, width, fits):
    """before anything is launched: with a wrapped sum CTAs would take rows that are not there.  (What fits goes on to the next check, that of
    the scratch.)"""
    stride = page * 2 * 64
    rc, text = call("ixb_attn_paged", requests=requests, rows=rows, hq=hq, q_stride=hq * 64, page=page, width=width, k_page_stride=stride, v_page_stride=stride,
                    scratch_bytes=4096)
    blocks = -(-rows * (hq // 2) // 8) * -(-width * page // 128)           # eight rows a group, the shortest blocks; at least
    assert rc == (4 if fits else 2) and fits == (blocks < 2**32), text
    assert fits or "too much" in text


def test_scratch_sizes():
    from ixrun_b200 import _lib

    f = _lib.lib().ixb_attn_paged_scratch_bytes
    assert f(96) == 0 and all(f(d) > 4096 for d in (64, 128, 256))


def test_host_tensors_are_refused():
    from ixrun_b200.logits import apply_rules
    from ixrun_b200.paged import page_release, page_step

    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        page_step(i(2), i(2), i(2, 3), i(4), i(1), 16, 5)
    with pytest.raises(ValueError):
        page_release(i(2).bool(), i(2), i(2, 3), i(4), i(1), 16)
    with pytest.raises(ValueError):
        apply_rules(torch.zeros(1, 64))


def test_ctypes_arguments_match_the_names_here():
    from ixrun_b200 import _lib

    for name, args in ARGS.items():
        types = getattr(_lib.lib(), name).argtypes
        assert len(types) == len(args), name
        for t, (key, value) in zip(types, args.items()):
            assert (t in (ctypes.c_float,)) == isinstance(value, float), (name, key)


def test_names_of_the_package():
    import ixrun_b200
    from ixrun_b200 import llama_runner, logits, paged

    for name in paged.__all__:
        assert getattr(ixrun_b200, name) is getattr(paged, name)
    assert ixrun_b200.apply_rules is logits.apply_rules
    assert ixrun_b200.PagedDecoder is llama_runner.PagedDecoder
    with pytest.raises(AttributeError):
        ixrun_b200.no_such_name


def host_account(lengths):
    """a PagedDecoder's account of its requests, without a model"""
    from ixrun_b200.llama_runner import PagedDecoder

    dec = PagedDecoder.__new__(PagedDecoder)
    n = len(lengths)
    dec.b, dec._known, dec._cached, dec._steps, dec._last, dec._came, dec._added = n, list(lengths), [0] * n, 0, [0] * n, list(range(n)), n
    return dec


@pytest.mark.parametrize("lengths", [(1,) * 8, (1, 1, 1, 40), (5, 9, 1, 30, 1, 1), (200, 100), (1,) * 20 + (7,) * 20])
@pytest.mark.parametrize("rows", [1, 2, 4, 7])
def test_no_request_of_a_paged_decoder_waits_for_good(lengths, rows):
    """Single tokens in turns, a prompt at least in every second step, prompts one after the other: all have answered twice after as many
    steps as that takes, with every second one for a prompt while there is one."""
    dec = host_account(lengths)
    answers = [0] * len(lengths)
    n = len(lengths)
    bound = 2 * sum(-(-p // rows) + 1 for p in lengths) + 4 * -(-n // rows) + 4
    for _ in range(bound):
        q = dec._share(rows)
        assert 0 < sum(q) <= rows and min(q) >= 0
        known = list(dec._known)
        dec._account(q)
        answers = [a + (x != y) for a, x, y in zip(answers, known, dec._known)]
    assert min(answers) >= 2


def test_rows_that_suffice_go_to_everybody():
    dec = host_account((1, 30, 1, 4))
    assert dec._share(100) == [1, 30, 1, 4]
    assert dec._share(10) == [1, 8, 1, 0] and dec._share(2) == [1, 0, 1, 0] and dec._share(1) == [1, 0, 0, 0]
    dec._account([1, 0, 1, 0])                         # the prompt that had nothing comes first
    assert dec._share(3) == [0, 3, 0, 0] and dec._share(40) == [1, 30, 1, 4]


@pytest.mark.parametrize("vocab,max_seq,max_bias", [(393217, 96, 4), (1000, 2**20 - 1, 4), (1000, 96, 2048), (1000, 96, -1)])
def test_a_paged_decoder_beyond_the_limits_of_its_rules_is_refused(vocab, max_seq, max_bias):
    """at the start, not in its first step, when tables and lengths have been written"""
    from types import SimpleNamespace

    from ixrun_b200.llama_runner import LlamaConfig, PagedDecoder

    cfg = LlamaConfig(n_layers=1, hidden=256, intermediate=512, n_heads=4, n_kv_heads=2, head_dim=64, vocab=vocab, max_seq=max_seq)
    with pytest.raises(ValueError):
        PagedDecoder(SimpleNamespace(weights="packed", glue="kernels", cfg=cfg), 2, 4, max_bias=max_bias)


def test_limits_of_the_rules_are_those_of_the_entry():
    from ixrun_b200 import logits

    v, n, k = logits.MAX_VOCAB, logits.MAX_TOKENS, logits.MAX_BIASES
    for changed in (dict(vocab=v + 1, pitch=v + 1, out_pitch=v + 1), dict(hist_len=n + 1, hist_pitch=n + 1), dict(n_bias=k + 1, bias_ids=P, bias_values=P)):
        assert call("ixb_logits", **changed)[0] == 2


def test_a_paged_decoder_is_captured_on_its_own_device(monkeypatch):
    """whatever device is current: streams, synchronisation and the capture are those of the decoder's"""
    from contextlib import contextmanager
    from types import SimpleNamespace

    from ixrun_b200.llama_runner import PagedDecoder

    at, seen = ["cuda:0"], []

    @contextmanager
    def device(d):
        at.append(d)
        yield
        at.pop()

    @contextmanager
    def on(*_):
        yield

    note = lambda what, result=None: lambda *_: (seen.append((what, at[-1])), result)[1]  # noqa: E731
    stream = SimpleNamespace(wait_stream=lambda _: None)
    for name, fake in (("device", device), ("stream", on), ("graph", on), ("Stream", note("stream", stream)), ("current_stream", note("current", stream)),
                       ("synchronize", note("synchronize")), ("CUDAGraph", note("graph", "graph"))):
        monkeypatch.setattr(torch.cuda, name, fake)
    dec = PagedDecoder.__new__(PagedDecoder)
    dec.b, dec._step, dec._bufs, dec._forward = 2, None, None, note("forward")
    dec.q_len = SimpleNamespace(device="cuda:1", zero_=lambda: None)
    assert dec.capture() is dec and dec.graph == "graph"
    assert [w for w, _ in seen].count("forward") == 3 and {d for _, d in seen} == {"cuda:1"}


@pytest.mark.parametrize("requests", [1, 8, 64])
def test_the_paged_figure_is_taken_behind_the_prompts(requests):
    """64 prompts of 128 tokens take more than four steps of 2048 rows, as the first answers come between"""
    from ixrun_b200.eval_llama import all_answering

    dec = host_account((128,) * requests)

    def step():
        q = dec._share(2048)
        known = list(dec._known)
        dec._account(q)
        return torch.tensor([1 if a != b else -1 for a, b in zip(known, dec._known)])

    dec.step = step
    all_answering(dec)
    assert all(k - c == 1 for k, c in zip(dec._known, dec._cached))
