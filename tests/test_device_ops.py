"""What the operators on device buffers refuse before they touch a GPU: the C
entry points' own checks (any non-null, aligned address will do: nothing is
read) and the tensor checks of laya_goish_b200.device."""
import ctypes

import pytest

from laya_goish_b200 import _lib

torch = pytest.importorskip("torch")

A = 4096  # an aligned non-null address


def invalid(rc, word):
    message = _lib.lib().laya_last_error().decode()
    assert rc == _lib.E_INVALID and word in message, (rc, message)


def cache(**change):
    f = dict(k=A, v=A, page_stride=8 * 64 * 64, head_stride=64 * 64, row_stride=64, pages=4, kv_heads=8, head_dim=64,
             type=1)
    f.update(change)
    return _lib.KvPages(**f)


def test_page_plan_arguments():
    L = _lib.lib()

    def plan(n=2, past=A, count=A, free=A, n_free=4, tables=A, stride=3, width=3, slots=A, pos=A, seqs=A, cap=5,
             offsets=A, lens=A, totals=A):
        return L.laya_page_plan(past, count, n, free, n_free, 0, tables, stride, width, slots, pos, seqs, cap, offsets,
                                lens, totals, None)

    invalid(plan(n=-1), "negative")
    invalid(plan(cap=-1), "negative")
    invalid(plan(width=-1), "negative")
    invalid(plan(n_free=-1), "negative")
    invalid(plan(stride=2), "overlap")
    invalid(plan(n=8193), "8192")
    for name in ("past", "count", "free", "tables", "slots", "offsets", "lens", "totals"):
        invalid(plan(**{name: None}), "null")
    for name in ("slots", "pos", "seqs"):
        invalid(plan(**{name: A + 8}), "aligned")


BAD_CACHES = [(dict(type=0), "F16 or BF16"), (dict(head_dim=96), "head_dim"), (dict(pages=0), "empty"),
              (dict(kv_heads=0), "empty"), (dict(row_stride=63), "strides"), (dict(page_stride=-8), "strides"),
              (dict(head_stride=1 << 38), "strides")]


@pytest.mark.parametrize("change,word", BAD_CACHES)
def test_caches(change, word):
    L = _lib.lib()
    c = cache(**change)
    invalid(L.laya_kv_append(ctypes.byref(c), 1, A, A, 512, 512, A, 1, None), word)
    invalid(L.laya_prefix_attention(ctypes.byref(c), ctypes.byref(_lib.PrefixArgs()), None), word)
    assert L.laya_prefix_attention_workspace(ctypes.byref(c), ctypes.byref(_lib.PrefixArgs())) == 0


def test_kv_append_arguments():
    L = _lib.lib()

    def append(c=None, kind=1, k=A, v=A, ks=512, vs=512, slots=A, rows=2):
        return L.laya_kv_append(ctypes.byref(c or cache()), kind, k, v, ks, vs, slots, rows, None)

    invalid(L.laya_kv_append(None, 1, A, A, 512, 512, A, 1, None), "null")
    invalid(append(kind=30), "cache's type")
    invalid(append(rows=-1), "negative")
    invalid(append(k=None), "null")
    invalid(append(slots=None), "null")
    invalid(append(cache(k=None)), "null")
    invalid(append(k=A + 8), "aligned")
    invalid(append(cache(v=A + 2)), "aligned")
    invalid(append(ks=516), "aligned")
    invalid(append(vs=504), "overlap")
    assert append(rows=0) == 0


def test_prefix_attention_arguments():
    L = _lib.lib()
    good = dict(q=A, q_stride=2048, rows=3, heads=32, offsets=A, n_seqs=2, max_q=2, prefix_pages=A, prefix_len=100,
                width=2, tables=A, table_stride=2, lens=A, scale=0.125, out=A, out_stride=2048, lse=None,
                workspace=None, workspace_bytes=0)

    def attend(c=None, **change):
        a = _lib.PrefixArgs(**dict(good, **change))
        return L.laya_prefix_attention(ctypes.byref(c or cache()), ctypes.byref(a), None)

    invalid(L.laya_prefix_attention(ctypes.byref(cache()), None, None), "null")
    for name in ("rows", "n_seqs", "max_q", "prefix_len", "width"):
        invalid(attend(**{name: -1}), "negative")
    invalid(attend(heads=12), "multiple of kv_heads")
    invalid(attend(cache(kv_heads=1), heads=129), "128")
    invalid(attend(rows=1 << 27), "too many")
    for x in (0.0, -1.0, float("nan"), float("inf")):
        invalid(attend(scale=x), "scale")
    for name in ("q", "out", "offsets", "lens", "prefix_pages", "tables"):
        invalid(attend(**{name: None}), "null")
    invalid(attend(q=A + 8), "16-byte")
    invalid(attend(out=A + 8), "16-byte")
    invalid(attend(q_stride=2044), "16 bytes")
    invalid(attend(q_stride=2040), "overlap")
    invalid(attend(out_stride=1024), "overlap")
    invalid(attend(table_stride=1), "overlap")
    for name in ("rows", "n_seqs", "max_q"):  # nothing to do
        assert attend(**{name: 0}) == 0


def test_token_logprobs_arguments():
    L = _lib.lib()

    def logprobs(kind=0, x=A, stride=50, rows=2, vocab=50, tokens=A, ts=1, c=1, top=2, lp=A, ids=A, tlp=A):
        return L.laya_token_logprobs(kind, x, stride, rows, vocab, tokens, ts, c, top, lp, None, None, ids, tlp, None)

    invalid(logprobs(kind=8), "F32, F16 or BF16")
    invalid(logprobs(rows=-1), "size")
    invalid(logprobs(vocab=0), "size")
    invalid(logprobs(c=-1), "size")
    invalid(logprobs(vocab=(1 << 30) + 1), "too large")
    invalid(logprobs(top=65), "top")
    invalid(logprobs(top=-1), "top")
    invalid(logprobs(stride=-1), "stride")
    invalid(logprobs(ts=-1), "stride")
    for name in ("x", "tokens", "lp", "ids", "tlp"):
        invalid(logprobs(**{name: None}), "null")
    invalid(logprobs(x=A + 2), "misaligned")
    invalid(logprobs(kind=1, x=A + 1), "misaligned")
    assert logprobs(rows=0) == 0
    invalid(L.laya_device_status(0, None), "null")


def test_prefix_attention_scale_stays_finite_in_log2_units():
    a = _lib.PrefixArgs(q=A, q_stride=2048, rows=3, heads=32, offsets=A, n_seqs=2, max_q=2, prefix_pages=A,
                        prefix_len=100, width=2, tables=A, table_stride=2, lens=A, scale=2.5e38, out=A, out_stride=2048)
    invalid(_lib.lib().laya_prefix_attention(ctypes.byref(cache()), ctypes.byref(a), None), "scale")


def test_score_arguments():
    L = _lib.lib()
    invalid(L.laya_score_tokens(None, A, A, 1, 0, A, None, None, None), "null model")


def test_host_tensors_are_refused():
    from laya_goish_b200 import device

    x = torch.zeros((2, 8))
    t = torch.zeros((2, 1), dtype=torch.int32)
    for call in (lambda: device.token_logprobs(x, t), lambda: device.KVPages(x, x),
                 lambda: device.page_plan(t[:, 0], t[:, 0], t[:, 0], t, 4), lambda: device.KVPages(None, None)):
        with pytest.raises(_lib.LayaError, match="CUDA tensor"):
            call()
    with pytest.raises(_lib.LayaError, match="KVPages"):
        device.kv_append(None, x, x, t)


def test_prefix_attention_refuses_keys_beyond_32_bit_positions():
    L = _lib.lib()
    good = dict(q=A, q_stride=2048, rows=3, heads=32, offsets=A, n_seqs=2, max_q=2, prefix_pages=A, prefix_len=100,
                width=2, tables=A, table_stride=1 << 30, lens=A, scale=0.125, out=A, out_stride=2048)
    most = (1 << 31) - 64
    for change in (dict(prefix_len=most + 1), dict(prefix_len=(1 << 31) - 1), dict(width=most // 64 + 1)):
        a = _lib.PrefixArgs(**dict(good, **change))
        invalid(L.laya_prefix_attention(ctypes.byref(cache()), ctypes.byref(a), None), "2^31 - 64 keys")
        assert L.laya_prefix_attention_workspace(ctypes.byref(cache()), ctypes.byref(a)) == 0
    a = _lib.PrefixArgs(**dict(good, prefix_len=most, width=most // 64, rows=0))
    assert L.laya_prefix_attention(ctypes.byref(cache()), ctypes.byref(a), None) == 0
