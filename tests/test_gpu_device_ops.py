"""The operators on CUDA tensors (laya_goish_b200.device) against plain 64-bit
implementations.

Tolerances count the roundings of each operator (u = eps / 2 of a type):
attention rounds each probability and each output to the cache's type, so an
output is within u (A + |o|) with A = sum_k p_k |v_k|; a score, a 32-bit sum
of head_dim products (each addition within 2^-23 in the tensor cores), moves a
probability by its own error; F16 probabilities below 2^-14 are within 2^-25
absolutely, and each joins at most n keys.  The log probabilities are 32-bit
sums of at most n / threads terms per thread joined in a tree."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    from laya_goish_b200 import _lib, device
    from laya_goish_b200._lib import LayaError

PAGE = 64
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def pages_of(n):
    return -(-n // PAGE)


def status_bits():
    import ctypes
    b = ctypes.c_uint32()
    _lib.check(_lib.lib().laya_device_status(0, ctypes.byref(b)))
    return b.value


@pytest.fixture(autouse=True)
def clean_status():
    status_bits()
    yield
    assert status_bits() == 0, "an operator flagged something that the test did not expect"


# ------------------------------------------------------------------ page plan

def plan_reference(past, count, free, tables, capacity, base):
    """(tables, slots, positions, seqs, offsets, lens, totals) by loops."""
    tables = tables.copy()
    n, width = tables.shape
    slots, pos, seqs = [-1] * capacity, [0] * capacity, [-1] * capacity
    offsets, lens, row, page = [], [], 0, 0
    for i in range(n):
        p, c = max(0, int(past[i])), max(0, int(count[i]))
        have, need = pages_of(p), min(pages_of(p + c), width)
        for a in range(have, need):
            tables[i, a] = free[page] if page < len(free) else -1
            page += 1
        offsets.append(min(row, capacity))
        lens.append(p + c)
        for t in range(c):
            if row < capacity:
                u = p + t
                pg = tables[i, u // PAGE] if u // PAGE < width else -1
                slots[row] = pg * PAGE + u % PAGE if pg >= 0 else -1
                pos[row], seqs[row] = base + u, i
            row += 1
    offsets.append(min(row, capacity))
    return tables, slots, pos, seqs, offsets, lens, [row, page]


def check_plan(past, count, free, tables, capacity, base=0):
    want = plan_reference(past, count, free, tables, capacity, base)
    t = torch.from_numpy(tables.copy()).cuda()
    got = device.page_plan(i32(past), i32(count), i32(free), t, capacity, base=base)
    for name, g, w in zip(("tables", "slots", "positions", "seqs", "offsets", "lens", "totals"),
                          (t, got.slots, got.positions, got.seqs, got.offsets, got.lens, got.totals), want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w).reshape(g.shape)), name


@pytest.mark.parametrize("n,most,seed", [(1, 1, 0), (1, 200, 1), (3, 65, 2), (31, 1, 3), (257, 130, 4), (513, 3, 5),
                                         (8192, 2, 6)])
@pytest.mark.parametrize("pad", [0, 7])
def test_page_plan(n, most, seed, pad):
    rng = np.random.default_rng(seed)
    past = rng.integers(0, 300, n)
    past[rng.random(n) < 0.3] = 0
    count = rng.integers(0, most + 1, n)
    need = [pages_of(p + c) for p, c in zip(past, count)]
    tables = rng.integers(0, 10 ** 6, (n, max(need) + 2)).astype(np.int32)
    check_plan(past.tolist(), count.tolist(), rng.permutation(sum(need) + 3).tolist(), tables,
               int(count.sum()) + pad, base=int(rng.integers(0, 1000)))


def test_page_plan_at_its_limits():
    tables = np.arange(12, dtype=np.int32).reshape(4, 3)
    # no sequences; nothing new; the list, the capacity and the table's width too short; negative values; page edges
    check_plan([], [], [1, 2], np.zeros((0, 3), np.int32), 5)
    check_plan([0, 5, 64, 128], [0, 0, 0, 0], [9], tables, 3)
    check_plan([0, 0, 0, 0], [64, 65, 1, 128], [7, 8, 9], tables, 300)
    check_plan([0, 60, 64, 100], [70, 10, 1, 30], list(range(20)), tables, 50)
    check_plan([190, 0, 500, 192], [10, 300, 4, 1], list(range(20)), tables, 320)
    check_plan([-5, 3, -1, 0], [4, -7, -2, 1], list(range(20)), tables, 6)
    check_plan([63, 64, 127, 128], [1, 1, 1, 1], [50, 51, 52, 53], tables, 4)
    check_plan([0, 0, 0, 0], [1, 2, 3, 4], [], tables, 10)
    check_plan([0, 0, 0, 0], [1, 2, 3, 4], [5] * 4, tables, 0)
    check_plan([1, 2], [1, 1], [3], np.zeros((2, 0), np.int32), 2)


def test_page_plan_strided_tables_and_repeat():
    wide = torch.full((3, 10), 77, dtype=torch.int32, device="cuda")
    view = wide[:, 2:6]
    past, count, free = i32([0, 64, 10]), i32([65, 1, 2]), i32([4, 5, 6])
    view[1, 0] = view[2, 0] = 9
    for _ in range(2):  # a second call over its own tables gives the same
        p = device.page_plan(past, count, free, view, 68)
        assert wide.cpu().tolist() == [[77, 77, 4, 5] + [77] * 6, [77, 77, 9, 6] + [77] * 6, [77, 77, 9] + [77] * 7]
        assert p.slots.cpu().tolist() == [4 * 64 + i for i in range(64)] + [5 * 64, 6 * 64, 9 * 64 + 10, 9 * 64 + 11]


# ------------------------------------------------------------------ append

def make_pages(pages, kv, hd, dtype, token_major, fill=None, gen=None):
    shape = (pages, PAGE, kv, hd) if token_major else (pages, kv, PAGE, hd)
    x = [torch.randn(shape, device="cuda", generator=gen).to(dtype) if fill is None else
         torch.full(shape, fill, device="cuda", dtype=dtype) for _ in range(2)]
    return [y.permute(0, 2, 1, 3) for y in x] if token_major else x


@pytest.mark.parametrize("kv,hd", [(1, 64), (8, 64), (3, 128), (2, 256), (40, 128)])
@pytest.mark.parametrize("dtype,src", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("token_major", [False, True])
def test_kv_append(kv, hd, dtype, src, token_major):
    g = torch.Generator(device="cuda").manual_seed(kv * hd)
    for rows in (1, 7, 130):
        k, v = make_pages(5, kv, hd, dtype, token_major, gen=g)
        wk, wv = k.clone(), v.clone()
        # rows of one projection's output: strided
        qkv = torch.randn((rows, 3, kv, hd), device="cuda", generator=g).to(src)
        nk, nv = qkv[:, 1], qkv[:, 2]
        slots = torch.randperm(5 * PAGE, device="cuda", generator=g)[:rows]
        slots[::5] = -1
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                wk[s // PAGE, :, s % PAGE] = nk[t].to(dtype)
                wv[s // PAGE, :, s % PAGE] = nv[t].to(dtype)
        device.kv_append(device.KVPages(k, v), nk, nv, slots)
        assert torch.equal(k, wk) and torch.equal(v, wv)


def test_kv_append_skips_and_flags_slots_outside():
    k, v = make_pages(2, 2, 64, F16, False, fill=3.0)
    new = torch.ones((4, 2, 64), device="cuda", dtype=F16)
    device.kv_append(device.KVPages(k, v), new, new, i64([-1, 128, -2, 1 << 40]))
    assert (k == 3).all() and (v == 3).all()
    with pytest.raises(LayaError, match="page or slot"):
        device.check_status()
    device.kv_append(device.KVPages(k, v), new[:0], new[:0], i64([]))


# ------------------------------------------------------------------ attention

def attend_reference(q, k, v, prefix_pages, prefix_len, tables, lens, new, scale):
    """64-bit outputs, lse and the tolerance of each, row by row of the batch."""
    rows, heads, hd = q.shape
    kv = k.shape[1]
    group = heads // kv
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    ltol = torch.zeros((rows, heads), dtype=torch.float64)

    def take(x, pages, n):
        return x[pages[:pages_of(n)].long()].double().cpu().transpose(0, 1).reshape(kv, -1, hd)[:, :n]

    kp, vp = take(k, prefix_pages, prefix_len), take(v, prefix_pages, prefix_len)
    first = 0
    for b, n in enumerate(new):
        own = int(lens[b])
        keys = torch.cat([kp, take(k, tables[b], own)], 1)
        vals = torch.cat([vp, take(v, tables[b], own)], 1)
        for j in range(n):
            see = prefix_len + max(0, own - n + j + 1)
            if see:
                x = q[first + j].double().cpu().view(kv, group, hd)
                s = torch.einsum("kgd,ksd->kgs", x, keys[:, :see]) * scale
                size = torch.einsum("kgd,ksd->kgs", x.abs(), keys[:, :see].abs()).amax(-1) * scale
                p = torch.softmax(s, -1)
                o = torch.einsum("kgs,ksd->kgd", p, vals[:, :see])
                a = torch.einsum("kgs,ksd->kgd", p, vals[:, :see].abs())
                ds = hd * 2.0 ** -23 * size + 2.0 ** -20
                t = u * (a + o.abs()) * 1.01 + a * 2 * ds[..., None]
                if q.dtype == F16:
                    t = t + see * 2.0 ** -25 * float(vals[:, :see].abs().max())
                    t = t + 2.0 ** -25  # an output below 2^-14
                out[first + j], tol[first + j] = o.view(heads, hd), t.view(heads, hd)
                e = torch.logsumexp(s, -1)
                lse[first + j] = e.view(-1)
                ltol[first + j] = (ds + 2.0 ** -22 * e.abs()).view(-1) + see * 2.0 ** -24
        first += n
    return out, tol, lse, ltol


class Batch:
    """Pages, tables and queries of a batch; what no row may see holds NaN."""

    def __init__(self, new, held, prefix, heads, kv, hd, dtype, token_major=False, pad=0, seed=0, poison=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)
        each = [pages_of(h) for h in held]
        pre = pages_of(prefix)
        total = pre + sum(each) + 2
        ids = rng.permutation(total).tolist()
        self.k, self.v = make_pages(total, kv, hd, dtype, token_major, gen=g)
        at, rows, used = pre, [], [(ids[:pre], prefix)]
        for e, h in zip(each, held):
            rows.append(ids[at:at + e] + [-1] * (max(each) + 1 - e))
            used.append((ids[at:at + e], h))
            at += e
        if poison:
            keep = torch.zeros((total, PAGE), dtype=torch.bool)
            for pages, n in used:
                for i, pg in enumerate(pages):
                    keep[pg, :min(PAGE, n - i * PAGE)] = True
            gone = ~keep.cuda()[:, None, :, None].expand(self.k.shape)
            self.k[gone] = math.nan
            self.v[gone] = math.inf
            self.v[..., ::2][gone[..., ::2]] = math.nan
        self.new, self.held, self.prefix = new, held, prefix
        self.prefix_pages, self.tables = i32(ids[:pre]), i32(rows)
        self.lens = i32(held)
        self.offsets = i32([0] + np.cumsum(new).tolist())
        self.rows = sum(new) + pad
        self.q = (1.5 * torch.randn((self.rows, heads, hd), device="cuda", generator=g)).to(dtype)
        self.pages = device.KVPages(self.k, self.v)
        self.scale = 1.0 / math.sqrt(hd)

    def run(self, max_q=None, q=None, out=None, lse=None, scale=None):
        q = self.q if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        lse = torch.full(q.shape[:2], 7.0, device="cuda") if lse is None else lse
        device.prefix_attention(q, self.pages, self.prefix_pages, self.prefix, self.tables, self.lens, self.offsets,
                                max(self.new) if max_q is None else max_q, scale=scale, out=out, lse=lse)
        return out, lse

    def check(self, out, lse, scale=None):
        want, tol, wl, lt = attend_reference(self.q, self.k, self.v, self.prefix_pages, self.prefix, self.tables,
                                             self.held, self.new, scale or self.scale)
        n = sum(self.new)
        d = (out[:n].double().cpu() - want[:n]).abs()
        assert not torch.isnan(d).any()
        assert (d <= tol[:n]).all(), f"{(d / tol[:n].clamp(min=1e-30)).max():.2f} of the tolerance"
        got = lse[:n].double().cpu()
        assert torch.equal(got == -math.inf, wl[:n] == -math.inf)
        fine = wl[:n] > -math.inf
        assert ((got - wl[:n]).abs()[fine] <= lt[:n][fine]).all()
        assert (out[n:] == 7).all() and (lse[n:] == 7).all()  # rows of no sequence


GEOMETRY = [(32, 8, 64), (7, 1, 128), (8, 2, 256), (4, 4, 64), (24, 2, 128), (33, 1, 64)]


@pytest.mark.parametrize("heads,kv,hd", GEOMETRY)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 400])
def test_attention_single_tokens(heads, kv, hd, dtype, prefix):
    held = [1, 64, 65, 200, 1, 130]
    b = Batch([1] * 6, held, prefix, heads, kv, hd, dtype, token_major=prefix % 2 == 1, seed=prefix + heads)
    b.check(*b.run())


@pytest.mark.parametrize("heads,kv,hd", GEOMETRY)
@pytest.mark.parametrize("prefix", [0, 100, 700])
def test_attention_ragged_suffixes(heads, kv, hd, prefix):
    # sequences without new tokens, without any, whose new rows are all they hold, padded rows behind
    b = Batch([5, 0, 19, 1, 70, 0], [5, 0, 150, 64, 70, 30], prefix, heads, kv, hd, F16, pad=9, seed=prefix + hd)
    b.check(*b.run())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,heads,kv,hd,prefix", [(1, 32, 8, 64, 3000), (3, 28, 4, 128, 2111), (40, 32, 8, 128, 1500),
                                                  (65, 8, 2, 256, 1000), (150, 12, 1, 64, 900)])
def test_attention_batches(n, heads, kv, hd, prefix, dtype):
    """Few and many rows per kv head, split and unsplit prefixes."""
    rng = np.random.default_rng(n)
    b = Batch([1] * n, rng.integers(1, 200, n).tolist(), prefix, heads, kv, hd, dtype, seed=n)
    b.check(*b.run())


# (new rows of each sequence, held tokens, prefix, heads, kv, hd): enough rows and
# prefix pages for the tensor-core kernel, with one and with two row tiles per
# CTA, row counts that leave a tile part empty, groups that do not divide 128
TENSOR_CORE = [
    ([1] * 60, [3] * 60, 2500, 32, 2, 64),
    ([5, 0, 40, 1, 3, 17], [5, 9, 200, 1, 64, 100], 4033, 33, 1, 64),
    ([1] * 61, list(range(1, 62)), 1345, 28, 4, 128),
    ([1] * 100, [1] * 100, 1250, 8, 2, 256),
    ([2] * 150, [2] * 150, 2048, 32, 8, 64),
    ([3] * 50, [70] * 50, 3001, 20, 4, 128),
    ([7, 0, 90], [7, 0, 90], 5000, 24, 2, 128),
    ([2] * 120, [5] * 120, 2900, 28, 4, 128),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", range(len(TENSOR_CORE)))
def test_attention_tensor_core_prefix(case, dtype):
    new, held, prefix, heads, kv, hd = TENSOR_CORE[case]
    b = Batch(new, held, prefix, heads, kv, hd, dtype, token_major=case % 2 == 1, pad=3 * (case % 3), seed=50 + case)
    out, lse = b.run()
    b.check(out, lse)
    again = b.run()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("case", [0, 3, 4, 5, 7])
def test_attention_tensor_core_extremes(case):
    """Rows whose maximum keeps growing along the keys, and single keys above all."""
    new, held, prefix, heads, kv, hd = TENSOR_CORE[case]
    b = Batch(new, held, prefix, heads, kv, hd, F16, seed=70 + case)
    b.q *= 8
    b.check(*b.run())
    # keys that grow along the prefix: O is rescaled again and again
    grow = torch.linspace(0.02, 4, pages_of(prefix), device="cuda")
    for i, pg in enumerate(b.prefix_pages.tolist()):
        b.k[pg] = b.k[pg] * grow[i].to(F16)
    b.check(*b.run())


def test_attention_tensor_core_pages_outside_the_cache():
    new, held, prefix, heads, kv, hd = TENSOR_CORE[0]
    b = Batch(new, held, prefix, heads, kv, hd, F16, seed=80, poison=False)
    pages = b.prefix_pages.clone()
    b.prefix_pages[3] = -7
    b.prefix_pages[20:22] = 1 << 29
    out, lse = b.run()
    assert status_bits() == 2
    keep = [i for i in range(pages_of(prefix)) if i not in (3, 20, 21)]
    want, tol, _, _ = attend_reference(b.q, b.k, b.v, pages[keep], prefix - 3 * 64, b.tables, held, new, b.scale)
    assert ((out.double().cpu() - want).abs() <= tol).all()
    # none at all: the own keys alone
    b.prefix_pages.fill_(-1)
    out, _ = b.run()
    assert status_bits() == 2
    want, tol, _, _ = attend_reference(b.q, b.k, b.v, pages, 0, b.tables, held, new, b.scale)
    assert ((out.double().cpu() - want).abs() <= tol).all()


def test_attention_long_own_keys_are_split():
    b = Batch([1, 1], [3000, 70], 0, 8, 2, 64, F16, seed=1)
    b.check(*b.run())
    b = Batch([2, 1], [2500, 1], 333, 8, 2, 128, BF16, seed=2)
    b.check(*b.run())
    b = Batch([40], [1500], 100, 8, 2, 64, F16, seed=3)
    b.check(*b.run())


def test_attention_without_keys_gives_zero():
    # new rows beyond the held tokens see nothing of their own; without a prefix nothing at all
    for prefix in (0, 70):
        b = Batch([3, 1, 2], [1, 0, 2], prefix, 8, 2, 64, F16, pad=2, seed=4)
        out, lse = b.run()
        b.check(out, lse)
        if not prefix:
            assert (out[:2] == 0).all() and (out[3] == 0).all() and (lse[:2] == -math.inf).all()


def test_attention_strided_rows_and_scale():
    b = Batch([2, 3, 1], [10, 80, 1], 150, 8, 2, 64, F16, seed=5)
    wide = torch.zeros((b.rows, 12, 64), device="cuda", dtype=F16)
    wide[:, 2:10] = b.q
    res = torch.full((b.rows, 16, 64), 7.0, device="cuda", dtype=F16)
    out, lse = b.run(q=wide[:, 2:10], out=res[:, 8:], scale=0.3)
    b.check(out, lse, scale=0.3)
    assert (res[:, :8] == 7).all()


def test_attention_extreme_scores():
    """One key far above all others, and rows of equal scores."""
    b = Batch([1, 1], [100, 65], 200, 8, 2, 64, F16, seed=6)
    b.q *= 20
    b.check(*b.run())
    b.q.zero_()
    b.check(*b.run())


def test_attention_pages_outside_the_cache_are_unseen():
    b = Batch([1, 1], [100, 65], 200, 8, 2, 64, F16, seed=7, poison=False)
    pages = b.prefix_pages.clone()
    b.prefix_pages[1] = 1 << 30
    b.tables[0, 1] = -1
    out, lse = b.run()
    assert status_bits() == 2
    # the same as a batch without those keys: prefix pages 0, 2, 3 and the first own page of sequence 0
    c = Batch([1, 1], [100, 65], 200, 8, 2, 64, F16, seed=7, poison=False)
    want, tol, _, _ = attend_reference(c.q, c.k, c.v, pages[[0, 2, 3]], 136, c.tables, [64, 65], [1, 1], c.scale)
    assert ((out.double().cpu() - want).abs() <= tol).all()


def test_attention_rows_beyond_max_q_and_lengths_beyond_the_table():
    b = Batch([3, 2], [64, 64], 100, 8, 2, 64, F16, seed=8)
    out, lse = b.run(max_q=2)
    assert status_bits() == 8
    full, _ = b.run()
    assert torch.equal(out[[0, 1, 3, 4]], full[[0, 1, 3, 4]]) and (out[2] == 7).all()
    b.lens[1] = 100000
    b.tables[:, 1] = b.tables[:, 0]
    b.run()
    assert status_bits() == 2


def test_attention_repeats_bitwise_on_streams_and_in_graphs():
    a = Batch([1] * 90, list(range(20, 110)), 1500, 32, 8, 64, F16, seed=9)  # tensor-core prefix
    b = Batch([4, 17], [40, 300], 130, 28, 4, 128, F16, seed=10)
    want = [a.run(), b.run()]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (s, x) in enumerate(zip(side, (a, b))):
            with torch.cuda.stream(s):
                got[i] = x.run()
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1])
    graphs, outs = [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(x.run())
        graphs.append(g)
    # replayed together on two streams, with new lengths written in between
    a.lens -= 3
    a.held = [h - 3 for h in a.held]
    want[0] = a.run()
    torch.cuda.synchronize()
    for _ in range(2):
        for s, g in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
    a.check(*outs[0])


# ------------------------------------------------------------------ log probabilities

def logprob_case(logits, tokens, top):
    got = device.token_logprobs(logits, tokens, top=top)
    x = logits.double().cpu()
    n, vocab = x.shape
    # relative to the maximum: lse = -1e30 + ln(50) has no room for the second term in 64 bits either
    most = x.amax(-1)
    fine = most > -math.inf
    d = x - torch.where(fine, most, torch.zeros_like(most))[:, None]
    ln = torch.log(torch.exp(d).sum(-1))
    lse = torch.where(fine, most + ln, most)
    y = d - torch.where(fine, ln, torch.zeros_like(ln))[:, None]
    p = torch.exp(y)
    # 32-bit sums of the terms of a thread, then a tree; |x - M| weighs the exponent's rounding
    rel = (vocab / 128 + 60) * 2.0 ** -24 + 2.0 ** -20
    there = torch.where(x > -math.inf, x, torch.zeros_like(x))
    far = (p * (there - there.amax(-1, keepdim=True)).abs()).nan_to_num(0).sum(-1) + 5

    def near(got, want, tol, what):
        got = got.double().cpu()
        assert torch.equal(got == -math.inf, want == -math.inf), what
        ok = want > -math.inf
        assert ((got - want).abs()[ok] <= tol.expand(want.shape)[ok]).all(), what

    tl = rel * far
    near(got.lse, lse, tl + lse.abs().nan_to_num(0, 0, 0) * 2.0 ** -22, "lse")
    ent = -torch.where(p > 0, p * y, torch.zeros_like(p)).sum(-1)
    near(got.entropy, torch.where(fine, ent, torch.zeros_like(ent)), 2 * tl * (1 + far), "entropy")
    t = tokens.long().cpu()
    inside = (t >= 0) & (t < vocab)
    want = torch.where(inside, y.gather(1, t.clamp(0, vocab - 1)), torch.zeros(t.shape, dtype=torch.float64))
    near(got.logprobs, want, tl[:, None] + want.abs().nan_to_num(0, 0, 0) * 2.0 ** -22 + 2.0 ** -20, "logprobs")
    if top:
        order = torch.sort(x + 0.0, dim=1, descending=True, stable=True)
        ids = torch.full((n, top), -1, dtype=torch.int64)
        lp = torch.full((n, top), -math.inf, dtype=torch.float64)
        m = min(top, vocab)
        ids[:, :m], lp[:, :m] = order.indices[:, :m], y.gather(1, order.indices[:, :m])
        ids[lp == -math.inf] = -1
        assert torch.equal(got.top_ids.long().cpu(), ids)
        near(got.top_logprobs, lp, tl[:, None] + lp.abs().nan_to_num(0, 0, 0) * 2.0 ** -22 + 2.0 ** -20, "top")
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 64, 65, 255, 300, 511, 1000, 4096, 8191, 32000, 65537, 152064])
def test_logprobs(vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for n, top in ((1, 20), (3, 64), (5, 1), (2, 0)):
        x = (2.5 * torch.randn((n, vocab), device="cuda", generator=g)).to(dtype)
        t = torch.randint(0, vocab, (n, 4), device="cuda", generator=g, dtype=torch.int32)
        t[:, 1] = -1
        logprob_case(x, t, top)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab,gap,shift", [(1000, 1, 0), (1000, 3, 5), (40001, 0, 1), (152064, 7, 3)])
def test_logprobs_unaligned_rows(vocab, gap, shift, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    wide = torch.full((5, vocab + gap + shift), 1e4, device="cuda", dtype=dtype)  # what lies between rows is not read
    wide[:, shift:shift + vocab] = (3 * torch.randn((5, vocab), device="cuda", generator=g)).to(dtype)
    t = torch.randint(0, vocab, (5, 9), device="cuda", generator=g, dtype=torch.int32)
    logprob_case(wide[:, shift:shift + vocab], t[:, 2:5], 10)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [50, 3000, 100000])
def test_logprobs_ties_masks_and_sorted_rows(vocab, dtype):
    low = torch.finfo(dtype).min
    rows = [torch.zeros(vocab), torch.full((vocab,), -2.5), torch.full((vocab,), -math.inf),
            torch.linspace(-8, 8, vocab), torch.linspace(8, -8, vocab)]
    ties = torch.zeros(vocab)
    ties[vocab // 2:] = 1.0
    rows.append(ties)
    few = torch.full((vocab,), -math.inf)
    few[vocab // 3], few[vocab - 1], few[0] = 1.0, 1.0, -3.0
    rows.append(few)
    rows.append(torch.where(torch.isinf(few), torch.tensor(low), few))  # the type's lowest value as the mask
    rows.append(torch.full((vocab,), low))
    zeros = torch.zeros(vocab)
    zeros[::2] = -0.0
    rows.append(zeros)
    big = torch.full((vocab,), -9.0)
    big[vocab - 20:] = torch.arange(20) / 4
    rows.append(big)
    x = torch.stack(rows).to(dtype).cuda()
    if dtype == F32:  # log softmax of the lowest value is itself: nothing left of the others' exponentials
        x[8] = -1e30
    t = i32([[0, vocab // 3, vocab - 1, -1]] * len(rows))
    for top in (1, 5, 20, 64):
        logprob_case(x, t, top)


def test_logprobs_nan_infinity_and_bad_tokens():
    x = torch.randn((4, 5000), device="cuda")
    x[0, 77], x[1, 4999], x[3, 5] = math.nan, math.inf, -math.inf
    t = i32([[1, -1, 2]] * 4)
    got = device.token_logprobs(x, t, top=3)
    for r in (0, 1):
        assert torch.isnan(got.lse[r]) and torch.isnan(got.entropy[r]) and torch.isnan(got.top_logprobs[r]).all()
        assert torch.isnan(got.logprobs[r, [0, 2]]).all() and got.logprobs[r, 1] == 0
        assert (got.top_ids[r] == -1).all()
    assert torch.isfinite(got.logprobs[2:]).all() and torch.isfinite(got.lse[2:]).all()
    device.check_status()
    got = device.token_logprobs(x[2:], i32([[5000], [-2]]))
    assert (got.logprobs == 0).all()
    with pytest.raises(LayaError, match="token id"):
        device.check_status()


def test_logprobs_many_rows_many_tokens_and_graph():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((700, 2000), device="cuda", generator=g).to(BF16)
    t = torch.randint(0, 2000, (700, 300), device="cuda", generator=g, dtype=torch.int32)
    want = logprob_case(x, t, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = device.token_logprobs(x, t, top=8)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert torch.equal(w, o)
    empty = device.token_logprobs(x[:0], t[:0], top=2)
    assert empty.top_ids.shape == (0, 2)
    assert device.token_logprobs(x[:2], t[:2, :0]).logprobs.shape == (2, 0)


# ------------------------------------------------------------------ together

def test_step_over_a_shared_prefix():
    """A step as it is used: plan, append, attend, log probabilities, twice (a
    prompt suffix each, then a token each), against a dense 64-bit model."""
    heads, kv, hd, vocab, prefix, n = 8, 2, 64, 3000, 150, 5
    g = torch.Generator(device="cuda").manual_seed(11)
    k, v = make_pages(24, kv, hd, F16, False, fill=math.nan)
    pages = device.KVPages(k, v)
    head = (torch.randn((heads * hd, vocab), device="cuda", generator=g) / 16).to(F16)
    free = torch.randperm(24, device="cuda", generator=g).int()
    # the prefix: a sequence of its own
    pre_table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    plan = device.page_plan(i32([0]), i32([prefix]), free, pre_table, prefix)
    dense = torch.randn((2, prefix, kv, hd), device="cuda", generator=g).to(F16)
    device.kv_append(pages, dense[0], dense[1], plan.slots)
    taken = int(plan.totals[1])
    assert taken == 3
    prefix_pages = pre_table[0, :3].contiguous()
    tables = torch.full((n, 3), -1, dtype=torch.int32, device="cuda")
    past = torch.zeros(n, dtype=torch.int32, device="cuda")
    own = [torch.zeros((2, 0, kv, hd), dtype=F16, device="cuda") for _ in range(n)]
    for counts in ([3, 63, 1, 80, 0], [1, 1, 1, 1, 1]):
        rows = sum(counts) + 2
        plan = device.page_plan(past, i32(counts), free[taken:].contiguous(), tables, rows, base=prefix)
        new = torch.randn((2, rows, kv, hd), device="cuda", generator=g)
        q = torch.randn((rows, heads, hd), device="cuda", generator=g).to(F16)
        device.kv_append(pages, new[0], new[1], plan.slots)
        out = device.prefix_attention(q, pages, prefix_pages, prefix, tables, plan.lens, plan.offsets, max(counts))
        logits = out.view(rows, -1) @ head
        tokens = torch.randint(0, vocab, (rows, 1), device="cuda", generator=g, dtype=torch.int32)
        got = logprob_case(logits, tokens, 5)
        assert got.top_ids.shape == (rows, 5)
        first = 0
        for b, c in enumerate(counts):
            own[b] = torch.cat([own[b], new[:, first:first + c].to(F16)], 1)
            first += c
        assert (out[first:] == 0).all()
        batch = [torch.cat([dense, o], 1).double().cpu() for o in own]
        first = 0
        for b, c in enumerate(counts):
            for j in range(c):
                see = prefix + own[b].shape[1] - c + j + 1
                x = q[first + j].double().cpu().view(kv, heads // kv, hd)
                p = torch.softmax(torch.einsum("kgd,skd->kgs", x, batch[b][0][:see]) / 8, -1)
                want = torch.einsum("kgs,skd->kgd", p, batch[b][1][:see]).reshape(heads, hd)
                a = torch.einsum("kgs,skd->kgd", p, batch[b][1][:see].abs()).reshape(heads, hd)
                d = (out[first + j].double().cpu() - want).abs()
                assert (d <= 2.0 ** -11 * (a + want.abs()) * 1.01 + a * 2.0 ** -12 + see * 2.0 ** -23).all()
                assert int(plan.positions[first + j]) == see - 1 and int(plan.seqs[first + j]) == b
            first += c
        taken += int(plan.totals[1])
        past = plan.lens


# ------------------------------------------------------------------ refusals

def test_refusals():
    b = Batch([1, 2], [64, 64], 100, 8, 2, 64, F16, seed=12)
    ok = dict(q=b.q, pages=b.pages, prefix_pages=b.prefix_pages, prefix_len=100, tables=b.tables, lens=b.lens,
              offsets=b.offsets, max_q=2)
    device.prefix_attention(**ok)

    def refused(word, **change):
        with pytest.raises(LayaError, match=word) as e:
            device.prefix_attention(**dict(ok, **change))
        assert e.value.code == _lib.E_INVALID

    refused("bfloat|float16", q=b.q.to(BF16))
    refused("head_dim", q=torch.zeros((3, 8, 128), device="cuda", dtype=F16))
    refused("multiple of kv_heads", q=b.q[:, :7])
    refused("contiguous", q=b.q.transpose(0, 1).contiguous().transpose(0, 1))
    refused("CUDA tensor", q=b.q.cpu())
    refused("hold prefix_len", prefix_len=129)
    refused("hold prefix_len", prefix_len=-1)
    refused("int32", lens=b.lens.long())
    refused("fit the sequences", offsets=b.offsets[:2].contiguous())
    refused("max_q", max_q=-1)
    refused("scale", scale=0.0)
    refused("scale", scale=math.nan)
    refused("scale", scale=math.inf)
    refused("q's shape", out=b.q[:2])
    refused("lse", lse=torch.zeros((3, 7), device="cuda"))
    refused("overlap", out=b.q[:1].expand(3, 8, 64))
    refused("forward only", q=b.q.clone().requires_grad_())
    shifted = torch.zeros(3 * 512 + 4, device="cuda", dtype=F16)[4:].view(3, 8, 64)
    refused("16-byte", q=shifted)
    refused("KVPages", pages=(b.k, b.v))

    def no_pages(word, k, v):
        with pytest.raises(LayaError, match=word):
            device.KVPages(k, v)

    no_pages("64 tokens", b.k[:, :, :32], b.v[:, :, :32])
    no_pages("F16 or BF16", b.k.float(), b.v.float())
    no_pages("head_dim", b.k[..., :32], b.v[..., :32])
    no_pages("same strides", b.k, b.v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3))
    no_pages("overlap", b.k[:1].expand(4, -1, -1, -1), b.v[:1].expand(4, -1, -1, -1))
    no_pages("same shape", b.k, b.v[:1])

    new = torch.zeros((2, 2, 64), device="cuda", dtype=F16)

    def no_append(word, k, v, slots):
        with pytest.raises(LayaError, match=word):
            device.kv_append(b.pages, k, v, slots)

    no_append("pages' type", new.to(BF16), new.to(BF16), i64([0, 1]))
    no_append("slot per row", new, new, i64([0]))
    no_append("int64", new, new, i32([0, 1]))
    no_append("overlap", new[:1].expand(2, 2, 64), new, i64([0, 1]))

    t = b.tables
    with pytest.raises(LayaError, match="one row per sequence"):
        device.page_plan(i32([1]), i32([1, 2]), i32([0]), t, 4)
    with pytest.raises(LayaError, match="capacity"):
        device.page_plan(i32([1, 1]), i32([1, 2]), i32([0]), t, -1)
    with pytest.raises(LayaError, match="8192"):
        z = torch.zeros(8193, dtype=torch.int32, device="cuda")
        device.page_plan(z, z, z, torch.zeros((8193, 1), dtype=torch.int32, device="cuda"), 4)

    x = torch.zeros((2, 50), device="cuda")
    with pytest.raises(LayaError, match="top"):
        device.token_logprobs(x, i32([[0], [0]]), top=65)
    with pytest.raises(LayaError, match="row per row"):
        device.token_logprobs(x, i32([[0]]))
    with pytest.raises(LayaError, match="F32, F16 or BF16"):
        device.token_logprobs(x.double(), i32([[0], [0]]))
    with pytest.raises(LayaError, match="int32"):
        device.token_logprobs(x, i64([[0], [0]]))
    with pytest.raises(LayaError, match="empty vocabulary"):
        device.token_logprobs(x[:, :0], i32([[0], [0]]))
    device.check_status()


# What a row may not see is not in its result, whatever its value: later tokens
# of its own sequence with NaN or infinite K and V, in both forms of the own-keys
# kernel (few rows per kv head, many), with and without a prefix.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nq,own,heads,kv,prefix", [(5, 9, 4, 2, 0), (5, 67, 4, 2, 100), (40, 40, 4, 1, 0),
                                                    (150, 170, 2, 2, 70), (16, 200, 8, 8, 0)])
def test_later_tokens_may_hold_anything(dtype, hd, nq, own, heads, kv, prefix):
    gen = torch.Generator().manual_seed(nq * own + hd)
    pages, width, pre = 12, (own + 63) // 64, (prefix + 63) // 64
    k = torch.randn(pages, kv, 64, hd, generator=gen).to(dtype).cuda()
    v = torch.randn(pages, kv, 64, hd, generator=gen).to(dtype).cuda()
    q = torch.randn(nq, heads, hd, generator=gen).to(dtype).cuda()
    order = torch.randperm(pages, generator=gen).to(torch.int32).cuda()
    prefix_pages, tables = order[:pre], order[pre:pre + width].reshape(1, width).contiguous()
    lens, offsets = torch.tensor([own], dtype=torch.int32).cuda(), torch.tensor([0, nq], dtype=torch.int32).cuda()

    def run():
        lse = torch.empty(nq, heads, dtype=torch.float32, device="cuda")
        return device.prefix_attention(q, device.KVPages(k, v), prefix_pages, prefix, tables, lens, offsets, nq,
                                       lse=lse), lse

    def place(tok):
        return int(tables[0, tok // 64]), tok % 64

    clean, clean_lse = run()
    for back, bad in ((1, float("nan")), (2, float("inf")), (nq // 2, float("-inf"))):
        first = nq - back  # the first row that sees the bad token
        page, at = place(own - back)
        saved = k[page, :, at].clone(), v[page, :, at].clone()
        v[page, :, at, ::3] = bad
        out, lse = run()
        assert torch.equal(out[:first], clean[:first]) and torch.equal(lse, clean_lse)
        seen = out[first:, :, ::3].float()
        # (an infinity times a probability that the type rounds to 0 is NaN)
        assert (seen.isnan() | (seen == bad)).all()
        assert torch.equal(out[first:, :, 1::3], clean[first:, :, 1::3])
        k[page, :, at] = bad
        out, lse = run()
        assert torch.equal(out[:first], clean[:first]) and torch.equal(lse[:first], clean_lse[:first])
        k[page, :, at], v[page, :, at] = saved
    device.check_status()


@pytest.mark.parametrize("rows,prefix", [(1, 70), (40, 200), (400, 3000)])
def test_a_query_that_is_not_a_number(rows, prefix):
    """NaN queries give NaN and leave the other rows alone (prefix kernels and join)."""
    gen = torch.Generator().manual_seed(rows)
    pages = (prefix + 63) // 64 + 1
    k = torch.randn(pages, 2, 64, 128, generator=gen).half().cuda()
    v = torch.randn(pages, 2, 64, 128, generator=gen).half().cuda()
    q = torch.randn(rows, 4, 128, generator=gen).half().cuda()
    order = torch.arange(pages, dtype=torch.int32).cuda()
    tables = torch.full((rows, 1), pages - 1, dtype=torch.int32).cuda()
    lens = torch.full((rows,), 3, dtype=torch.int32).cuda()
    offsets = torch.arange(rows + 1, dtype=torch.int32).cuda()
    res = []
    for i in range(2):
        if i:
            q[rows // 2, 1] = float("nan")
        lse = torch.empty(rows, 4, dtype=torch.float32, device="cuda")
        out = device.prefix_attention(q, device.KVPages(k, v), order[:-1], prefix, tables, lens, offsets, 1, lse=lse)
        res.append((out, lse))
    device.check_status()
    (a, al), (b, bl) = res
    hit = torch.zeros(rows, 4, dtype=torch.bool, device="cuda")
    hit[rows // 2, 1] = True
    assert b[hit].isnan().all() and bl[hit].isnan().all()
    assert torch.equal(a[~hit], b[~hit]) and torch.equal(al[~hit], bl[~hit])


# Few rows over a long prefix: many partial results per row, which the join
# shares out (both prefix kernels, a count that leaves the last group idle).
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,prefix,heads,kv,hd", [([1], 2500, 4, 1, 64), ([1, 1, 1], 7000, 10, 2, 128),
                                                    ([2, 0, 1], 2177, 4, 2, 256), ([1] * 33, 6000, 8, 2, 256),
                                                    ([20], 6400, 7, 1, 64), ([1] * 5, 16000, 16, 1, 128)])
def test_attention_many_partial_results(new, prefix, heads, kv, hd, dtype):
    held = [n + 40 * (i % 3) for i, n in enumerate(new)]
    b = Batch(new, held, prefix, heads, kv, hd, dtype, pad=2, seed=prefix)
    b.check(*b.run())


# A logit of -inf is a token that is not there, whatever the others hold: rows
# of the type's lowest value (a mask) and -inf (padding of the vocabulary) alone,
# short, long and cut over a cluster, the rows' starts aligned and not.  n equal
# logits: log probability -ln n, entropy ln n.  The sum is n times one number,
# which is within 2^-22 of e^(x - M) (ex2.approx), added up within n / 128 + 60
# roundings in a row; ln and the sums with it round a few times more.
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab,there", [(50, 1), (1000, 999), (3001, 64), (32000, 1000), (152064, 70000)])
@pytest.mark.parametrize("rows", [1, 40, 700])
def test_logprobs_lowest_values_beside_minus_infinity(rows, vocab, there, dtype):
    low = torch.finfo(dtype).min
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    for gap in (0, 3):
        x = torch.full((rows, vocab + gap), -math.inf, device="cuda", dtype=dtype)[:, gap:]
        ids = torch.stack([torch.randperm(vocab, device="cuda", generator=g)[:there] for _ in range(min(rows, 4))])
        ids = ids[torch.arange(rows, device="cuda") % ids.shape[0]].sort(-1).values
        x.scatter_(1, ids, low)
        t = torch.stack([ids[:, 0], ids[:, -1]], 1).int()
        got = device.token_logprobs(x, t, top=5)
        ln = math.log(there)
        tol = (there / 128 + 60) * 2.0 ** -24 + 2.0 ** -22 + 8 * 2.0 ** -24 * (1 + ln)
        assert (got.logprobs.double() + ln).abs().max() <= tol
        assert (got.entropy.double() - ln).abs().max() <= tol
        assert (got.lse.double() - (low + ln)).abs().max() <= tol + abs(low) * 2.0 ** -23
        k = min(5, there)
        assert torch.equal(got.top_ids[:, :k].long(), ids[:, :k]) and (got.top_ids[:, k:] == -1).all()
        assert (got.top_logprobs[:, :k].double() + ln).abs().max() <= tol
        assert (got.top_logprobs[:, k:] == -math.inf).all()


def check_logprob_rows(x, tokens, top=0):
    """Outputs against 64 bits with tolerances that know no offset of the row.
    y = (x - M) log2 e has two roundings at most (2^-24 of it each, and log2 e
    itself is 2^-26 off), so a term is within 2^-22 (ex2.approx) + 3 |y| 2^-24
    of its size; M is at most 6 below the maximum.  A sum of them adds
    vocab / 128 roundings in a row and, where M moves and states are joined, at
    most 60 more (a factor ex2.approx each); ln, products and sums with the
    results add a few units of theirs.  lse has the offset and one rounding."""
    u = 2.0 ** -24
    got = device.token_logprobs(x, tokens, top=top)
    x = x.double().cpu()
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    s = e.sum(-1)
    p = e / s[:, None]
    far = (p * torch.where(p > 0, d.abs(), torch.zeros_like(d))).sum(-1) + 6  # mean |y| ln 2, at most
    rel = (x.shape[1] / 128 + 60) * u + 2.0 ** -22 + 6 * far * u  # of the sum, so absolutely of its ln
    ln = torch.log(s)
    y = d - ln[:, None]
    mean = torch.where(p > 0, p * d, torch.zeros_like(d)).sum(-1)
    assert ((got.entropy.double().cpu() - (ln - mean)).abs() <= 2 * rel * (1 + far) + 8 * u * (ln + far)).all()
    want = y.gather(1, tokens.long().cpu())
    tol = rel[:, None] + 8 * u * (want.abs() + ln[:, None] + 6)
    assert ((got.logprobs.double().cpu() - want).abs() <= tol).all()
    lse = x.amax(-1) + ln
    assert ((got.lse.double().cpu() - lse).abs() <= rel + 8 * u * (ln + 6) + 2 * u * lse.abs()).all()
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_ids.long().cpu(), order)
        want = y.gather(1, order)
        assert ((got.top_logprobs.double().cpu() - want).abs() <= rel[:, None] + 8 * u * (want.abs() + ln[:, None] + 6)).all()


# A common offset of a row changes nothing but lse.
@pytest.mark.parametrize("about", [20, -20, 3000, -3000, 30000, -30000, 64000])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (3, 32000), (500, 32000)])
def test_logprobs_with_a_common_offset(rows, vocab, about):
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = about + 2.5 * torch.randn((rows, vocab), device="cuda", generator=g)
    x[1] = about + torch.linspace(-30, 20, vocab, device="cuda")  # the reference moves again and again
    check_logprob_rows(x, torch.randint(0, vocab, (rows, 2), device="cuda", generator=g, dtype=torch.int32), top=4)


# Rows about large values: masked throughout (-1e10), or logits that big; about
# the values where the arithmetic changes; up to the type's ends.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("about", [65000, -65000, 1e5, -1e6, 1e9, 1e10, -1e10, -1e20, 9e29, -1e30, 3e38, -3e38])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (3, 32000), (500, 32000)])
def test_logprobs_far_from_zero(rows, vocab, about, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = about + 2.5 * torch.randn((rows, vocab), device="cuda", generator=g)
    x[0] = about  # all the same
    x[1, ::3] = 0.0  # beside ordinary ones
    x[2, 1::2] = -math.inf
    x[2, ::5] = torch.finfo(dtype).min
    t = torch.randint(0, vocab, (rows, 2), device="cuda", generator=g, dtype=torch.int32)
    t[2] = 2  # one that is there
    check_logprob_rows(x.to(dtype), t, top=4)


def test_status_bits_set_while_the_word_is_read_are_not_lost():
    """One thread reads the status word again and again, with a token bit to
    clear each time; another sets the page bit 2000 times, at some place of a
    reading, and waits until a reading has it."""
    import random
    import sys
    import threading
    import time

    k, v = make_pages(1, 1, 64, F16, False, fill=0.0)
    pages, row, outside = device.KVPages(k, v), torch.ones((1, 1, 64), device="cuda", dtype=F16), i64([1 << 20])
    x, bad = torch.zeros((1, 8), device="cuda"), i32([[99]])
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    seen, stop = [0], threading.Event()

    def reader():
        while not stop.is_set():
            with torch.cuda.stream(side[1]):
                device.token_logprobs(x, bad)
            seen[0] |= status_bits() & 2

    t = threading.Thread(target=reader)
    t.start()
    lost, r, interval = 0, random.Random(1), sys.getswitchinterval()
    try:
        sys.setswitchinterval(1e-6)  # both threads run all the while
        for _ in range(2000):
            until = time.perf_counter() + 3e-4 * r.random()
            while time.perf_counter() < until:
                pass
            seen[0] = 0
            with torch.cuda.stream(side[0]):
                device.kv_append(pages, row, row, outside)
            side[0].synchronize()
            until = time.monotonic() + 2
            while not seen[0] and time.monotonic() < until:
                pass
            if not seen[0]:
                lost += 1
                break
    finally:
        sys.setswitchinterval(interval)
        stop.set()
        t.join()
        status_bits()
    assert not lost


# max_q is a bound: one as loose as a context length, or the largest there is,
# changes neither results nor what is accepted.
@pytest.mark.parametrize("bound", [7, 70, 100000, 2 ** 31 - 1])
@pytest.mark.parametrize("new,prefix", [([1, 1, 1], 0), ([1, 1, 1], 130), ([3, 0, 1], 700), ([70, 2], 100)])
def test_attention_with_a_loose_bound_of_rows(new, prefix, bound):
    b = Batch(new, [n + 50 for n in new], prefix, 8, 2, 64, F16, pad=3, seed=prefix + len(new))
    b.check(*b.run(max_q=max(bound, max(new))))


@pytest.mark.parametrize("rows", [1, 2, 40])
def test_attention_of_the_widest_groups_with_the_largest_bound(rows):
    b = Batch([1] * rows, [9] * rows, 70, 128, 1, 64, F16, seed=rows)
    b.check(*b.run(max_q=2 ** 31 - 1))


def test_no_gradient_is_dropped_without_a_word():
    """Pages that require a gradient, and forward-mode tangents anywhere, are refused like other inputs with gradients."""
    from torch.autograd import forward_ad

    b = Batch([1, 2], [64, 64], 100, 8, 2, 64, F16, seed=13)
    new, slots = torch.zeros((2, 2, 64), device="cuda", dtype=F16), i64([0, 1])
    x, t = torch.zeros((2, 50), device="cuda"), i32([[0], [0]])
    for name in ("k", "v"):
        kv = dict(k=b.k.clone(), v=b.v.clone())
        kv[name].requires_grad_()
        pages = device.KVPages(kv["k"], kv["v"])
        b.pages = pages
        with pytest.raises(LayaError, match="forward only"):
            b.run()
        with pytest.raises(LayaError, match="forward only"):
            device.kv_append(pages, new, new, slots)
        with torch.no_grad():
            b.run()
            device.kv_append(pages, new, new, slots)
    pages = b.pages = device.KVPages(b.k, b.v)
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(y, torch.ones_like(y)) for y in (b.q, new, x)]
        with pytest.raises(LayaError, match="tangent"):
            b.run(q=dual[0])
        for k, v in ((dual[1], new), (new, dual[1])):
            with pytest.raises(LayaError, match="tangent"):
                device.kv_append(pages, k, v, slots)
        with pytest.raises(LayaError, match="tangent"):
            device.token_logprobs(dual[2], t)
        b.pages = device.KVPages(forward_ad.make_dual(b.k, torch.ones_like(b.k)), b.v)
        with pytest.raises(LayaError, match="tangent"):
            b.run()
    device.check_status()


def test_writes_are_seen_by_autograd():
    """What a call writes in place cannot go unnoticed into a backward pass that saved it before."""
    b = Batch([1, 2], [64, 64], 100, 8, 2, 64, F16, seed=14)
    new, slots = torch.ones((2, 2, 64), device="cuda", dtype=F16), i64([0, 1])
    out, lse = torch.zeros_like(b.q), torch.zeros((b.rows, 8), device="cuda")

    def plan():
        device.page_plan(i32([64, 64]), i32([1, 2]), i32([0, 1]), b.tables, 3)

    for call, tensors in ((lambda: b.run(out=out, lse=lse), (out, lse)),
                          (lambda: device.kv_append(b.pages, new, new, slots), (b.k, b.v)), (plan, (b.tables,))):
        for t in tensors:
            before = t._version
            call()
            assert t._version == before + 1
            if t.is_floating_point():
                w = torch.ones((), device="cuda", requires_grad=True)
                loss = (w * t).float().sum()
                call()
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    loss.backward()
    with torch.inference_mode():  # inference tensors have no version
        q = b.q.clone()
        b.run(q=q, out=torch.zeros_like(q))
    device.check_status()


def test_pages_whose_tensors_moved_are_refused():
    for name in ("k", "v"):
        b = Batch([1, 2], [64, 64], 100, 8, 2, 64, F16, seed=15)
        t = getattr(b, name)
        old = t.data  # keeps the old memory alive
        new, slots = torch.ones((2, 2, 64), device="cuda", dtype=F16), i64([0, 1])
        t.data = old.clone()
        with pytest.raises(LayaError, match="moved"):
            b.run()
        with pytest.raises(LayaError, match="moved"):
            device.kv_append(b.pages, new, new, slots)
        b.pages = device.KVPages(b.k, b.v)
        b.check(*b.run())


def prefix_kernel(rows, heads, kv, hd, prefix):
    """(row tiles per CTA of the tensor-core kernel or 0 for the other one, row
    tiles), by the rules that the launch code states."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    group, pages = heads // kv, pages_of(prefix)
    small = -(-rows * group // 16)
    if rows * group <= 16 or small * kv * pages * (hd // 64) ** 2 <= 10 * sms:
        return 0, small
    tiles = -(-rows // (128 // group))
    return (1 if hd == 256 or tiles * kv * pages <= 16 * sms else 2), tiles


# Two row tiles per CTA and an odd number of them, so that the last CTAs have
# one; the widest groups (a tile of one token, rows of a tile unused).
ODD_TILES = [
    ([1] * 330, 2048, 32, 8, 64),
    ([11] * 31, 4300, 12, 4, 64),
    ([1] * 230, 2900, 28, 4, 128),
    ([3, 5, 200, 0, 110], 3001, 20, 4, 128),
    ([1] * 21, 8000, 128, 1, 64),
    ([1] * 24, 6400, 100, 1, 128),
    ([2, 3], 4000, 65, 1, 256),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", range(len(ODD_TILES)))
def test_attention_tensor_core_odd_tiles_and_wide_groups(case, dtype):
    new, prefix, heads, kv, hd = ODD_TILES[case]
    pad = case % 2
    nt, tiles = prefix_kernel(sum(new) + pad, heads, kv, hd, prefix)
    assert nt == (1 if hd == 256 else 2) and tiles % 2 == 1
    b = Batch(new, [n + i % 5 for i, n in enumerate(new)], prefix, heads, kv, hd, dtype, token_major=case % 2 == 0,
              pad=pad, seed=90 + case)
    out, lse = b.run()
    b.check(out, lse)
    again = b.run()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_the_tensor_core_cases_reach_both_forms():
    forms = {hd: set() for hd in (64, 128, 256)}
    for new, _, prefix, heads, kv, hd in TENSOR_CORE:
        nt, _ = prefix_kernel(sum(new), heads, kv, hd, prefix)
        assert nt
        forms[hd].add(nt)
    assert forms == {64: {1, 2}, 128: {1, 2}, 256: {1}}


@pytest.mark.parametrize("new,held,prefix,heads,kv,hd", [([700], [700], 0, 8, 2, 64), ([513, 1, 1], [600, 90, 1], 70, 4, 2, 128),
                                                         ([257, 0, 300], [257, 5, 1000], 300, 2, 2, 256),
                                                         ([40, 2], [50, 2], 0, 128, 1, 64)])
def test_attention_of_prompts(new, held, prefix, heads, kv, hd):
    """Many new rows, alone and beside single ones."""
    b = Batch(new, held, prefix, heads, kv, hd, BF16, pad=1, seed=len(new) + hd)
    b.check(*b.run())


def test_no_memory_for_the_outputs_is_torch_s_own_error():
    n = 1 << 30  # rows that share their memory; 64 alternatives of each would take 0.5 TB
    with pytest.raises(torch.cuda.OutOfMemoryError):
        device.token_logprobs(torch.zeros((1, 8), device="cuda").expand(n, 8), i32([[0]]).expand(n, 1), top=64)
    device.check_status()
