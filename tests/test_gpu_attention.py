"""GPU: head norms with rotation, append to a paged cache and attention over it, against 64-bit forms on the CPU.
Tolerances are the bounds of attn_ref.py."""
import ctypes
import pathlib
import subprocess
import sys

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-6
NAN = float("nan")


def close(got, want, bound):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (int(bad.sum()), float((err / bound)[bad].max()), bad.nonzero()[0].tolist())


def randn(*shape, seed, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).to(torch.bfloat16).cuda()


def freqs(rotary, base):
    return [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]


def no_device_error():
    from helios_b200 import _lib
    assert _lib.device_error() == 0


class Step:
    """A batch over a cache whose unused slots and pages hold NaN; pages in random order."""

    def __init__(self, q_lens, kv_lens, hk, d, page, seed, *, order="hsd", behind=0, before=0, spare=2, poison=NAN,
                 window=0):
        from helios_b200 import attention as A
        g = torch.Generator().manual_seed(seed)
        used = [-(-n // page) for n in kv_lens]
        n_pages = sum(used) + spare
        perm = torch.randperm(n_pages, generator=g)
        self.table = torch.full((len(kv_lens), max(1, max(used))), -7, dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = perm[at:at + u]
            at += u
        k = torch.full((n_pages, hk, page, d), poison)
        v = torch.full((n_pages, hk, page, d), poison)
        for b, n in enumerate(kv_lens):
            for p in range(used[b]):
                m = min(page, n - p * page)
                k[self.table[b, p], :, :m] = torch.randn(hk, m, d, generator=g)
                v[self.table[b, p], :, :m] = torch.randn(hk, m, d, generator=g)
        if window:      # pages that lie before every query's window were given back: their entries are stale
            for b, n in enumerate(kv_lens):
                gone = max(0, n - q_lens[b] - window + 1) // page
                for p in range(min(gone, used[b])):
                    k[self.table[b, p]], v[self.table[b, p]] = poison, poison
                    self.table[b, p] = -1
        self.kc, self.vc = k.to(torch.bfloat16), v.to(torch.bfloat16)
        if order == "shd":      # [pages, slots, heads, head_dim] storage
            kd, vd = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (self.kc, self.vc))
        elif order == "layers":  # one layer's slice of a tensor that holds three
            big = torch.full((2, n_pages, 3, hk, page, d), NAN, dtype=torch.bfloat16, device="cuda")
            big[0, :, 1], big[1, :, 1] = self.kc.cuda(), self.vc.cuda()
            kd, vd = big[0, :, 1], big[1, :, 1]
        else:
            kd, vd = self.kc.cuda(), self.vc.cuda()
        self.cache = A.PagedKVCache(kd, vd)
        self.q_offsets = [before + sum(q_lens[:b]) for b in range(len(q_lens) + 1)]
        self.kv_lens, self.rows = kv_lens, before + sum(q_lens) + behind
        self.t_off = torch.tensor(self.q_offsets, dtype=torch.int32, device="cuda")
        self.t_kv = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        self.t_table = self.table.cuda()
        self.batch = A.PagedBatch(self.t_off, self.t_kv, self.t_table, max_q=max(max(q_lens), 1))

    def reference(self, q, scale, window):
        return R.attention(q.cpu(), self.kc, self.vc, self.q_offsets, self.kv_lens, self.table.tolist(), scale, window)


# ---- norms with rotation -------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,hq,hk,d,rotary,base,first", [
    (1, 16, 8, 256, 256, 10000.0, 16383),
    (1, 1, 1, 64, 16, 10000.0, 0),
    (3, 5, 3, 64, 64, 1e6, 262000),
    (7, 3, 1, 128, 64, 10000.0, 2 ** 31 - 8),
    (5, 16, 1, 512, 128, 1e6, 14336),
    (2, 3, 2, 512, 384, 10000.0, 77),
    (2, 4, 1, 512, 512, 10000.0, 131071),
    (700, 16, 8, 256, 128, 10000.0, 5),
    (611, 32, 8, 128, 128, 1e6, 100000),
])
def test_qk_norm_rope(cuda, tokens, hq, hk, d, rotary, base, first):
    from helios_b200 import attention as A
    row = randn(tokens, (hq + 2 * hk) * d, seed=tokens, std=1.7)
    q, k = row[:, : hq * d].unflatten(1, (hq, d)), row[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    wq, wk = randn(d, seed=1, std=0.1, mean=1), randn(d, seed=2, std=0.1, mean=1)
    pos = torch.arange(first, first + tokens, dtype=torch.int32)
    rope = A.Rope(d, base, rotary_dim=rotary)
    before = row.clone()
    qo, ko = A.qk_norm_rope(q, k, pos.cuda(), rope, wq, wk, eps=EPS)
    torch.cuda.synchronize()
    assert torch.equal(row, before)
    for x, w, got in ((q, wq, qo), (k, wk, ko)):
        close(got, *R.norm_rope(x.cpu(), pos, freqs(rotary, base), rotary, w.cpu(), EPS))
    # in place on the matmul's rows: the same bits, and the values untouched
    A.qk_norm_rope(q, k, pos.cuda(), rope, wq, wk, eps=EPS, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(row[:, (hq + hk) * d:], before[:, (hq + hk) * d:])


def test_qk_norm_rope_without_weights_scaled_positions_and_zero_rows(cuda):
    from helios_b200 import attention as A
    d = 256
    q, k = randn(9, 2, d, seed=3), randn(9, 1, d, seed=4)
    q[3] = 0                                     # a zero row stays zero
    pos = torch.tensor([0, -1, 5, 6, 7, 100000, 3, 2, 1], dtype=torch.int32)
    f = [0.125 * x for x in freqs(d, 10000.0)]
    f[5] = 0.0
    rope = A.Rope(d, inv_freq=f)
    qo, ko = A.qk_norm_rope(q, k, pos.cuda(), rope, eps=EPS)
    close(qo, *R.norm_rope(q.cpu(), pos, f, d, None, EPS))
    close(ko, *R.norm_rope(k.cpu(), pos, f, d, None, EPS))
    assert not qo[3].any()
    e = torch.empty(0, 2, d, dtype=torch.bfloat16, device="cuda")
    A.qk_norm_rope(e, e[:, :1], torch.empty(0, dtype=torch.int32, device="cuda"), rope)


# ---- append ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("q_lens,kv_lens,hq,hk,d,rotary,page,order", [
    ([1], [1], 2, 1, 64, 64, 16, "hsd"),
    ([1, 1, 1], [17, 16, 300], 16, 8, 256, 256, 16, "shd"),
    ([5, 0, 33, 1], [5, 9, 70, 64], 4, 2, 128, 64, 32, "layers"),
    ([64, 200], [1000, 200], 16, 1, 512, 128, 64, "hsd"),
    ([3] * 40, [3 + 11 * i for i in range(40)], 2, 1, 256, 256, 128, "hsd"),
])
@pytest.mark.parametrize("norm_values", [True, False])
def test_kv_append(cuda, q_lens, kv_lens, hq, hk, d, rotary, page, order, norm_values):
    from helios_b200 import attention as A
    s = Step(q_lens, kv_lens, hk, d, page, 5, order=order, before=1, behind=3)
    row = randn(s.rows, (hq + 2 * hk) * d, seed=6, std=1.7)
    q, k, v = (row[:, a * d: b * d].unflatten(1, (b - a, d)) for a, b in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
    wq, wk = randn(d, seed=1, std=0.1, mean=1), randn(d, seed=2, std=0.1, mean=1)
    rope = A.Rope(d, 10000.0, rotary_dim=rotary)
    q_out = torch.full((s.rows, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    got = A.kv_append(q, k, v, s.cache, s.batch, rope, wq, wk, eps=EPS, norm_values=norm_values, q_out=q_out)
    assert got is q_out
    no_device_error()
    toks = R.tokens(s.q_offsets, kv_lens)
    r = torch.tensor([t[0] for t in toks])
    pos = torch.tensor([t[2] for t in toks])
    f = freqs(rotary, 10000.0)
    close(q_out[r], *R.norm_rope(q.cpu()[r], pos, f, rotary, wq.cpu(), EPS))
    rest = torch.ones(s.rows, dtype=torch.bool)
    rest[r] = False
    assert (q_out.cpu()[rest] == 7.0).all()      # rows of no sequence
    page_id = torch.tensor([int(s.table[b, p // page]) for _, b, p in toks])
    slot = torch.tensor([p % page for _, _, p in toks])
    kc, vc = s.cache.k.cpu(), s.cache.v.cpu()
    close(kc[page_id, :, slot], *R.norm_rope(k.cpu()[r], pos, f, rotary, wk.cpu(), EPS))
    if norm_values:
        want = R.norm(v.cpu()[r], None, EPS)
        close(vc[page_id, :, slot], want, R.half_step(want) + 2.0 ** -19 * want.abs())
    else:
        assert torch.equal(vc[page_id, :, slot], v.cpu()[r])
    # every other slot keeps its bits
    keep = torch.ones(kc.shape[0], page, dtype=torch.bool)
    keep[page_id, slot] = False
    for now, was in ((kc, s.kc), (vc, s.vc)):
        assert torch.equal(now.transpose(1, 2)[keep].view(torch.int16), was.transpose(1, 2)[keep].view(torch.int16))


def test_kv_append_shared_key_and_value_without_queries(cuda):
    from helios_b200 import attention as A
    s = Step([3, 1], [40, 16], 1, 512, 16, 8)
    k = randn(4, 1, 512, seed=9)
    rope = A.Rope(512, 1e6, rotary_dim=128)
    assert A.kv_append(None, k, k, s.cache, s.batch, rope, eps=EPS) is None
    no_device_error()
    toks = R.tokens(s.q_offsets, s.kv_lens)
    pos = torch.tensor([t[2] for t in toks])
    page_id = torch.tensor([int(s.table[b, p // 16]) for _, b, p in toks])
    close(s.cache.k.cpu()[page_id, :, pos % 16], *R.norm_rope(k.cpu(), pos, freqs(128, 1e6), 128, None, EPS))
    want = R.norm(k.cpu(), None, EPS)
    close(s.cache.v.cpu()[page_id, :, pos % 16], want, R.half_step(want) + 2.0 ** -19 * want.abs())


# ---- attention -------------------------------------------------------------------------------------------

def check_attention(q_lens, kv_lens, hq, hk, d, page, window, *, scale=None, order="hsd", seed=11, behind=0, before=0):
    from helios_b200 import attention as A
    s = Step(q_lens, kv_lens, hk, d, page, seed, order=order, behind=behind, before=before, window=window)
    q = randn(s.rows, hq, d, seed=seed + 1)
    attend = A.PagedAttention(hq, hk, d)
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((s.rows, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    attend(q, s.cache, s.batch, scale=scale, window=window, out=out)
    no_device_error()
    want, bound = s.reference(q, scale, window)
    mine = ~torch.isnan(want).any(-1).any(-1)
    close(out.cpu()[mine], want[mine], bound[mine])
    assert (out.cpu()[~mine] == 7.0).all()
    again = attend(q, s.cache, s.batch, scale=scale, window=window)
    assert torch.equal(again[mine.cuda()], out[mine.cuda()])       # the same bits every time
    return s, q, attend, out


@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 1023, 4100])
def test_attention_one_token(cuda, kv):
    check_attention([1], [kv], 4, 2, 256, 16, 0)


@pytest.mark.parametrize("d,hq,hk", [(64, 12, 4), (64, 1, 1), (128, 32, 8), (256, 16, 8), (256, 2, 1), (512, 16, 1), (512, 3, 1)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attention_tokens_of_a_ragged_batch(cuda, d, hq, hk, page):
    check_attention([1] * 7, [1, 333, 64, 1500, 128, 17, 700], hq, hk, d, page, 0)


@pytest.mark.parametrize("d,hq,hk,n", [(256, 16, 8, 8), (256, 16, 8, 15), (256, 4, 1, 16), (512, 16, 1, 2), (512, 16, 1, 4),
                                       (128, 32, 8, 5), (64, 7, 1, 9), (64, 64, 1, 1)])
@pytest.mark.parametrize("window", [0, 100])
def test_attention_drafted_blocks(cuda, d, hq, hk, n, window):
    check_attention([n] * 3, [n, n + 190, 515 + n], hq, hk, d, 32, window, behind=2, before=1)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 1024])
def test_attention_window_one_token(cuda, window):
    check_attention([1, 1, 1], [1, 64, 1333], 4, 2, 256, 16, window)


@pytest.mark.parametrize("d,hq,hk", [(64, 12, 4), (128, 32, 8), (256, 16, 8), (256, 1, 1)])
@pytest.mark.parametrize("q_lens,kv_lens,window", [([1], [65], 0), ([1], [1536], 0), ([1], [1537], 0), ([2, 0, 1], [700, 0, 3], 0),
                                                   ([1, 3, 1, 2], [5000, 3, 1100, 900], 1024), ([1, 1], [0, 500], 0)])
def test_attention_few_units_of_few_tiles(cuda, d, hq, hk, q_lens, kv_lens, window):
    if 0 not in kv_lens or q_lens[kv_lens.index(0)] == 0:
        check_attention(q_lens, kv_lens, hq, hk, d, 64, window, behind=1)
        return
    from helios_b200 import _lib
    from helios_b200 import attention as A
    s = Step(q_lens, kv_lens, hk, d, 64, 11)                  # more new tokens than keys: reported, zeros
    q = randn(s.rows, hq, d, seed=12)
    out = A.PagedAttention(hq, hk, d)(q, s.cache, s.batch)
    assert _lib.device_error() == _lib.ERR_LENS
    close(out, *s.reference(q, d ** -0.5, 0))
    assert not out[0].any() and out[1].any()


def test_a_row_of_nan_scores_is_nan(cuda):
    """A query that is NaN has no maximum: its row is NaN, the others are not; few units, many, and a chunk."""
    from helios_b200 import attention as A
    for q_lens, kv_lens in (([1, 1], [300, 200]), ([1, 1], [5000, 200]), ([100], [300])):
        s = Step(q_lens, kv_lens, 2, 128, 16, 61)
        q = randn(s.rows, 4, 128, seed=62)
        q[1, 2] = NAN
        out = A.PagedAttention(4, 2, 128)(q, s.cache, s.batch)
        assert out[1, 2].isnan().all()
        out[1, 2], q[1, 2] = 0, 0
        assert not out.isnan().any()
        no_device_error()


@pytest.mark.parametrize("order", ["shd", "layers"])
def test_attention_cache_orders(cuda, order):
    check_attention([1, 3], [90, 200], 8, 4, 128, 32, 0, order=order)


@pytest.mark.parametrize("n", [1, 90])
def test_attention_window_as_long_as_the_table(cuda, n):
    """Windows that hide nothing, up to the largest."""
    from helios_b200 import attention as A
    s = Step([n], [200], 2, 128, 16, 7)
    q = randn(n, 4, 128, seed=8)
    attend = A.PagedAttention(4, 2, 128)
    want = attend(q, s.cache, s.batch)
    for window in (200, 208, 5000, 2 ** 31 - 1):
        assert torch.equal(attend(q, s.cache, s.batch, window=window), want)


def test_attention_shared_prefix_pages_and_max_kv(cuda):
    """Two sequences over the same pages, and a table wider than the step's lengths."""
    from helios_b200 import attention as A
    s = Step([3, 2], [100, 100], 2, 128, 16, 9)
    s.table[1] = s.table[0]
    s.t_table.copy_(s.table)
    q = randn(5, 4, 128, seed=8)
    wide = torch.full((2, 400), -1, dtype=torch.int32, device="cuda")
    wide[:, :7] = s.t_table
    attend = A.PagedAttention(4, 2, 128)
    for batch in (s.batch, A.PagedBatch(s.t_off, s.t_kv, wide, max_q=3), A.PagedBatch(s.t_off, s.t_kv, wide, max_q=3, max_kv=100)):
        out = attend(q, s.cache, batch)
        no_device_error()
        close(out, *s.reference(q, 128 ** -0.5, 0))


def test_attention_peaked_scores(cuda):
    check_attention([1, 2], [900, 300], 16, 1, 512, 64, 0, scale=1.0)


def test_attention_many_sequences(cuda):
    """More sequences than a warp has lanes, some without new tokens, and more units than CTAs."""
    n = 150
    check_attention([i % 3 for i in range(n)], [max(i % 3, 5 * i % 211) for i in range(n)], 8, 4, 64, 16, 0)


@pytest.mark.parametrize("d,hq,hk", [(64, 12, 4), (128, 8, 8), (256, 4, 2), (256, 3, 1), (512, 16, 1), (512, 2, 1)])
@pytest.mark.parametrize("n,kv,page,window", [(128, 128, 64, 0), (130, 130, 16, 0), (200, 331, 32, 0), (65, 1000, 128, 0),
                                              (257, 900, 16, 100), (300, 301, 64, 1), (90, 700, 256, 517)])
def test_attention_chunk(cuda, d, hq, hk, n, kv, page, window):
    check_attention([n], [kv], hq, hk, d, page, window)


@pytest.mark.parametrize("d,hq,hk,window", [(256, 16, 8, 0), (512, 16, 1, 0), (128, 6, 2, 200), (64, 64, 1, 0)])
def test_attention_mixed_batch(cuda, d, hq, hk, window):
    """Prompts of several lengths beside single tokens and drafted blocks, an empty sequence, and padding rows."""
    check_attention([150, 1, 0, 33, 8, 1, 200], [150, 700, 9, 33, 300, 1, 450], hq, hk, d, 16, window, before=3, behind=5)


def test_attention_chunk_split_over_a_long_context(cuda):
    """Few row tiles: their keys are split over CTAs, some of which have none in the short sequence."""
    check_attention([100, 100], [2500, 101], 2, 1, 256, 64, 0)
    check_attention([100, 100], [3000, 101], 2, 1, 512, 64, 150)
    check_attention([16, 16], [3000, 17], 16, 1, 512, 64, 0)


@pytest.mark.parametrize("d,hq,hk", [(64, 12, 4), (128, 12, 4), (256, 6, 2), (512, 3, 1)])
def test_attention_chunk_same_bits_whatever_ran_before(cuda, d, hq, hk):
    """Three heads a group: 42 tokens of a tile leave two spare rows, which hold what the call before left in shared
    memory. Large queries of four heads a group are that call."""
    from helios_b200 import attention as A
    s = Step([300, 77], [900, 400], hk, d, 32, 71)
    q = randn(s.rows, hq, d, seed=72)
    attend, other = A.PagedAttention(hq, hk, d), A.PagedAttention(4 * hk, hk, d)
    want = None
    for i in range(12):
        large = randn(s.rows, 4 * hk, d, seed=80 + i, std=4.0 ** (i % 4))
        other(large, s.cache, s.batch, scale=1.0)
        got = attend(q, s.cache, s.batch, scale=1.0)
        want = got if want is None else want
        assert torch.equal(got, want), i
    no_device_error()


def test_attention_chunk_peaked_scores(cuda):
    check_attention([150], [500], 16, 1, 512, 64, 0, scale=1.0)


def test_attention_chunk_cache_orders_and_strides(cuda):
    for order in ("shd", "layers"):
        check_attention([140, 3], [190, 200], 8, 4, 128, 32, 0, order=order)
    from helios_b200 import attention as A
    s = Step([100], [150], 2, 128, 16, 21)
    big = randn(100, 6 + 4, 128, seed=22)
    q = big[:, :6]
    out = torch.zeros(6, 100, 128, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    A.PagedAttention(6, 2, 128)(q, s.cache, s.batch, out=out)
    no_device_error()
    close(out, *s.reference(q, 128 ** -0.5, 0))


def test_attention_rows_that_see_nothing(cuda):
    """A sequence without keys, and one with more new tokens than keys (refused for the append, reported)."""
    from helios_b200 import _lib
    from helios_b200 import attention as A
    s = Step([1, 3, 2], [40, 0, 1], 2, 128, 16, 3)
    q = randn(6, 4, 128, seed=4)
    out = A.PagedAttention(4, 2, 128)(q, s.cache, s.batch)
    assert _lib.device_error() == _lib.ERR_LENS
    want, bound = s.reference(q, 128 ** -0.5, 0)
    close(out, want, bound)
    assert not out[1:5].any() and out[5].any()
    s = Step([140, 80, 70], [60, 0, 300], 2, 128, 16, 3)      # the same for the chunk kernel
    q = randn(290, 4, 128, seed=4)
    out = A.PagedAttention(4, 2, 128)(q, s.cache, s.batch)
    assert _lib.device_error() == _lib.ERR_LENS
    close(out, *s.reference(q, 128 ** -0.5, 0))
    assert not out[:80].any() and not out[140:220].any() and out[80].any()


def test_attention_strided_queries_and_output(cuda):
    from helios_b200 import attention as A
    s = Step([2, 1], [77, 300], 2, 128, 16, 21)
    big = randn(3, 4 + 4, 128, seed=22)
    q = big[:, :4]                                            # a slice of the q|k|v rows
    out = torch.zeros(4, 3, 128, dtype=torch.bfloat16, device="cuda").transpose(0, 1)    # head-major
    A.PagedAttention(4, 2, 128)(q, s.cache, s.batch, out=out)
    no_device_error()
    close(out, *s.reference(q, 128 ** -0.5, 0))


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 2], [130, 64]), ([100], [130])])
def test_offsets_beyond_32_bits(cuda, q_lens, kv_lens):
    """Pages 2^31 elements apart and token rows 2^25 or 2^30 apart: append and attention of few rows and of a chunk."""
    from helios_b200 import attention as A
    d, hk, hq, page, pages = 64, 2, 4, 64, 4
    n = sum(q_lens)
    apart = 2 ** 30 if n < 4 else 2 ** 25
    big = torch.empty(3 * 2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    strides = (2 ** 31, page * d, d, 1)
    kd = big.as_strided((pages, hk, page, d), strides, 0)
    vd = big.as_strided((pages, hk, page, d), strides, 2 ** 16)
    q = big.as_strided((n, hq, d), (apart, d, 1), 2 ** 17)
    k, v = (big.as_strided((n, hk, d), (apart, d, 1), 2 ** 17 + i * 2 ** 12) for i in (1, 2))
    out = big.as_strided((n, hq, d), (apart, d, 1), 2 ** 17 + 3 * 2 ** 12)
    s = Step(q_lens, kv_lens, hk, d, page, 51, spare=0)
    for i in range(s.kc.shape[0]):                     # the cache's pages, from the far end
        kd[pages - 1 - i], vd[pages - 1 - i] = s.kc[i].cuda(), s.vc[i].cuda()
    s.t_table.copy_(torch.where(s.table >= 0, pages - 1 - s.table, -1))
    fresh = [randn(n, h, d, seed=52 + i) for i, h in enumerate((hq, hk, hk))]
    for to, x in zip((q, k, v), fresh):
        to.copy_(x)
    cache, rope = A.PagedKVCache(kd, vd), A.Rope(d)
    attend = A.PagedAttention(hq, hk, d)
    A.kv_append(q, k, v, cache, s.batch, rope, q_out=q)
    attend(q, cache, s.batch, out=out)
    want_q = A.kv_append(*fresh, s.cache, A.PagedBatch(s.t_off, s.t_kv, s.table.cuda(), max_q=max(q_lens)), rope)
    assert torch.equal(q, want_q)
    for b, (m, far) in enumerate(zip(kv_lens, s.t_table.tolist())):
        for p in range(-(-m // page)):
            near, held = int(s.table[b, p]), min(page, m - p * page)
            assert torch.equal(kd[far[p], :, :held], s.cache.k[near, :, :held])
            assert torch.equal(vd[far[p], :, :held], s.cache.v[near, :, :held])
    s.kc, s.vc = s.cache.k.cpu(), s.cache.v.cpu()
    close(out, *s.reference(want_q, d ** -0.5, 0))
    no_device_error()


def test_page_ids_and_lengths_outside_are_reported_and_touch_nothing(cuda):
    from helios_b200 import _lib
    from helios_b200 import attention as A
    d, hk, hq = 64, 1, 2
    rope = A.Rope(d)
    k = randn(2, hk, d, seed=1)
    for bad in (-1, 1 << 30, 5):
        s = Step([1, 1], [20, 33], hk, d, 16, 2, spare=0)     # 5 pages: ids 0..4
        s.t_table[1, 2] = bad
        A.kv_append(None, k, k, s.cache, s.batch, rope)
        assert _lib.device_error() == _lib.ERR_PAGE
        changed = (s.cache.k.cpu().view(torch.int16) != s.kc.view(torch.int16)).flatten(1).any(1)
        assert changed.sum() == 1 and changed[s.table[0, 1]]
        out = A.PagedAttention(hq, hk, d)(randn(2, hq, d, seed=3), s.cache, s.batch)
        assert _lib.device_error() == _lib.ERR_PAGE
        assert torch.isfinite(out[0]).all()
    for off, kv, code in (([0, 1, 2], [20, 4000], _lib.ERR_TABLE), ([0, 2, 1], [20, 33], _lib.ERR_LENS),
                          ([0, 1, 9], [20, 33], _lib.ERR_LENS), ([0, 1, 2], [20, -4], _lib.ERR_LENS),
                          ([-1, 1, 2], [20, 33], _lib.ERR_LENS)):
        s = Step([1, 1], [20, 33], hk, d, 16, 2, spare=0)
        s.t_off.copy_(torch.tensor(off, dtype=torch.int32))
        s.t_kv.copy_(torch.tensor(kv, dtype=torch.int32))
        A.kv_append(None, k, k, s.cache, s.batch, rope)
        assert _lib.device_error() == code
        A.PagedAttention(hq, hk, d)(randn(2, hq, d, seed=3), s.cache, s.batch)
        assert _lib.device_error() == code
    no_device_error()


def test_chunk_bad_pages_and_lengths(cuda):
    from helios_b200 import _lib
    from helios_b200 import attention as A
    attend = A.PagedAttention(2, 1, 64)
    q = randn(200, 2, 64, seed=3)
    for bad in (-1, 1 << 30, 15):
        s = Step([100, 100], [100, 120], 1, 64, 16, 2, spare=0)
        s.t_table[1, 2] = bad
        out = attend(q, s.cache, s.batch)
        assert _lib.device_error() == _lib.ERR_PAGE
        want, bound = s.reference(q, 0.125, 0)
        close(out[:100], want[:100], bound[:100])
    for off, kv, code in (([0, 100, 200], [100, 4000], _lib.ERR_TABLE), ([0, 150, 100], [100, 120], _lib.ERR_LENS),
                          ([0, 100, 999], [100, 120], _lib.ERR_LENS), ([0, 100, 200], [100, -9], _lib.ERR_LENS)):
        s = Step([100, 100], [100, 120], 1, 64, 16, 2, spare=0)
        s.t_off.copy_(torch.tensor(off, dtype=torch.int32))
        s.t_kv.copy_(torch.tensor(kv, dtype=torch.int32))
        attend(q, s.cache, s.batch)
        assert _lib.device_error() == code
    no_device_error()


def test_refusals(cuda):
    from helios_b200 import _lib
    from helios_b200 import attention as A
    s = Step([1], [20], 2, 128, 16, 1)
    q = randn(1, 4, 128, seed=1)
    attend = A.PagedAttention(4, 2, 128)
    for bad in (float("nan"), 0.0, -1.0):
        with pytest.raises(ValueError, match="scale"):
            attend(q, s.cache, s.batch, scale=bad)
    for bad in (-1, 2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="window"):
            attend(q, s.cache, s.batch, window=bad)
    with pytest.raises(ValueError, match="out must not be q"):
        attend(q, s.cache, s.batch, out=q)
    with pytest.raises(ValueError, match="token_stride"):
        attend(q.expand(3, 4, 128), s.cache, s.batch)
    with pytest.raises(ValueError, match="max_q"):
        A.PagedBatch(s.t_off, s.t_kv, s.t_table, max_q=0)
    with pytest.raises(ValueError, match="must hold 2"):
        A.PagedBatch(s.t_off[:1], s.t_kv, s.t_table, max_q=1)
    with pytest.raises(ValueError, match="query heads"):
        attend(q[:, :2], s.cache, s.batch)
    with pytest.raises(ValueError, match="heads are not the handle's"):
        A.PagedAttention(4, 4, 128)(q, s.cache, s.batch)
    with pytest.raises(ValueError, match=r"\[tokens, heads, 128\]"):
        attend(q[:, :, :64], s.cache, s.batch)
    with pytest.raises(ValueError, match="bfloat16"):
        attend(q.float(), s.cache, s.batch)
    with pytest.raises(ValueError, match="contiguous, strides"):
        attend(randn(1, 4, 132, seed=1)[:, :, 4:], s.cache, s.batch)
    with pytest.raises(ValueError, match="rows overlap"):
        q2 = randn(2, 4, 128, seed=1)
        attend(q2, s.cache, s.batch, out=q2[:1].expand(2, 4, 128))
    with pytest.raises(_lib.G4qError, match="power of two"):
        t = torch.zeros(3, 2, 24, 128, dtype=torch.bfloat16, device="cuda")
        attend(q, A.PagedKVCache(t, t), s.batch)
    rope = A.Rope(64)
    with pytest.raises(ValueError, match=r"\[tokens, heads, 64\]"):
        A.qk_norm_rope(q, q, torch.zeros(1, dtype=torch.int32, device="cuda"), rope)
    with pytest.raises(ValueError, match="head_dim is not the rope's"):
        k = randn(1, 2, 64, seed=1)
        A.kv_append(None, k, k, s.cache, s.batch, rope)
    with pytest.raises(ValueError, match="one entry per token"):
        k = randn(2, 2, 64, seed=1)
        A.qk_norm_rope(k, k, torch.zeros(1, dtype=torch.int32, device="cuda"), rope)
    rope.free()
    with pytest.raises(ValueError, match="freed"):
        rope.handle
    attend.free()
    with pytest.raises(ValueError, match="freed"):
        attend(q, s.cache, s.batch)


@pytest.mark.parametrize("tokens", [1, 3])
def test_outputs_that_overlap_inputs(cuda, tokens):
    """Views of one buffer qualify while no element is shared; anything else is refused before a launch."""
    from helios_b200 import attention as A
    d, hq, hk = 64, 4, 2
    rope = A.Rope(d)
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    base = randn(tokens, 2 * hq + 2 * hk, d, seed=1)
    q, k = base[:, :hq].clone(), base[:, hq:hq + hk].clone()
    want_q, want_k = A.qk_norm_rope(q, k, pos, rope)

    def run(views):
        buf = base.clone()
        flat = torch.zeros(tokens * (2 * hq + 2 * hk) * d + 64, dtype=torch.bfloat16, device="cuda")
        qv, kv, qo, ko = views(buf, flat)
        qv.copy_(q), kv.copy_(k)
        got = A.qk_norm_rope(qv, kv, pos, rope, q_out=qo, k_out=ko)
        assert torch.equal(got[0], want_q) and torch.equal(got[1], want_k)

    # behind each other in a token's row, in place, heads in turn, heads outside of the tokens
    run(lambda b, f: (b[:, :hq], b[:, hq:hq + hk], b[:, hq + hk:2 * hq + hk], b[:, 2 * hq + hk:]))
    run(lambda b, f: (b[:, :hq], b[:, hq:hq + hk], b[:, :hq], b[:, hq:hq + hk]))
    run(lambda b, f: (b[:, 0:2 * hq:2], b[:, 2 * hq:2 * hq + hk], b[:, 1:2 * hq:2], b[:, 2 * hq + hk:]))
    run(lambda b, f: (f[:tokens * hq * d].view(hq, tokens, d).transpose(0, 1), b[:, :hk],
                      f[tokens * hq * d:2 * tokens * hq * d].view(hq, tokens, d).transpose(0, 1), b[:, hk:2 * hk]))
    # a head on, half a head on, the other one's rows, the other output's rows
    bad = [lambda b, f: (b[:, :hq], b[:, 2 * hq:2 * hq + hk], b[:, 1:hq + 1], b[:, 2 * hq + hk:]),
           lambda b, f: (f[:tokens * hq * d].view(tokens, hq, d), b[:, :hk],
                         f[32:tokens * hq * d + 32].view(tokens, hq, d), b[:, hk:2 * hk]),
           lambda b, f: (b[:, :hq], b[:, hq:hq + hk], b[:, hq:2 * hq], b[:, 2 * hq:2 * hq + hk]),
           lambda b, f: (b[:, :hq], b[:, hq:hq + hk], b[:, 2 * hk + hq:], b[:, hq + hk + 1:hq + 2 * hk + 1]),
           lambda b, f: (b[:, :hq], b[:, hq:hq + hk], b[:, :hq], b[:, :hk])]
    for views in bad:
        with pytest.raises(ValueError, match="overlaps other rows"):
            run(views)

    s = Step([tokens], [20], hk, d, 16, 1)
    attend = A.PagedAttention(hq, hk, d)
    want = attend(q, s.cache, s.batch)
    buf = base.clone()
    buf[:, :hq].copy_(q)
    assert torch.equal(attend(buf[:, :hq], s.cache, s.batch, out=buf[:, hq:2 * hq]), want)
    with pytest.raises(ValueError, match="out must not be q"):
        attend(buf[:, :hq], s.cache, s.batch, out=buf[:, 1:hq + 1])
    no_device_error()


def test_chunk_of_one_query_head_without_a_head_stride(cuda):
    """The stride of a single head is not used: zero qualifies at the C interface, for a chunk as for few rows."""
    from helios_b200 import _lib
    from helios_b200 import attention as A
    s = Step([100], [130], 1, 64, 16, 2)
    q, out = randn(100, 1, 64, seed=3), torch.zeros(100, 1, 64, dtype=torch.bfloat16, device="cuda")
    attend = A.PagedAttention(1, 1, 64)
    rows = [_lib.G4qHeadRows(t.data_ptr(), 64, 0, 1) for t in (q, out)]
    _lib.call("g4q_paged_attention", attend.handle, ctypes.byref(rows[0]), 100, ctypes.byref(s.cache.c),
              ctypes.byref(s.batch._view(16)), 0.125, 0, ctypes.byref(rows[1]), torch.cuda.current_stream().cuda_stream)
    close(out, *s.reference(q, 0.125, 0))


def test_first_calls_inside_a_capture(cuda):
    """A process whose first calls are captured: nothing of theirs needs a run before."""
    code = """
import torch
from helios_b200 import _lib, attention as A
torch.manual_seed(0)
def make(n, kv):
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return A.PagedBatch(t([0, n]), t([kv]), t([list(range(16))]), max_q=n)
rope, attend, cache = A.Rope(128), A.PagedAttention(4, 2, 128), A.PagedKVCache.allocate(16, 32, 2, 128)
cache.k.normal_(), cache.v.normal_()
q, k, v = (torch.randn(150, h, 128, device="cuda").bfloat16() for h in (4, 2, 2))
few, many = make(2, 500), make(150, 400)
def step():
    return [attend(A.kv_append(q[:n], k[:n], v[:n], cache, b, rope), cache, b) for n, b in ((2, few), (150, many))]
g = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    out = step()
g.replay()          # appends: from here on the cache holds the same keys before and after a step
want = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, want)) and _lib.device_error() == 0
"""
    root = pathlib.Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_step_replays_in_a_cuda_graph_with_new_lengths(cuda):
    """append + attention captured once, replayed as the sequences grow: the lengths and tables are read on the
    device. Two graphs of one stream share the handle's scratch."""
    from helios_b200 import attention as A
    hq, hk, d, page = 4, 2, 128, 16
    s = Step([1, 1], [400, 50], hk, d, page, 31, spare=3, poison=0.0)
    rope, attend = A.Rope(d), A.PagedAttention(hq, hk, d)
    q, k, v = (randn(2, h, d, seed=32 + h) for h in (hq, hk, hk))
    t_kv = torch.tensor([100, 20], dtype=torch.int32, device="cuda")
    batch = A.PagedBatch(s.t_off, t_kv, s.t_table, max_q=1)
    qo, out, out2 = (torch.zeros(2, hq, d, dtype=torch.bfloat16, device="cuda") for _ in range(3))

    def step(o):
        A.kv_append(q, k, v, s.cache, batch, rope, q_out=qo)
        attend(qo, s.cache, batch, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for o in (out, out2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(o)
        graphs.append(g)
    for lens in ([101, 21], [102, 22], [399, 50], [1, 1]):
        t_kv.copy_(torch.tensor(lens, dtype=torch.int32))
        out.zero_(), out2.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        s.kc, s.vc = s.cache.k.cpu(), s.cache.v.cpu()
        s.kv_lens = lens
        close(out, *s.reference(qo, d ** -0.5, 0))
        assert torch.equal(out, out2)
    no_device_error()
    del graphs


def test_side_stream_and_empty_step(cuda):
    from helios_b200 import attention as A
    s = Step([1], [33], 2, 64, 16, 41)
    q = randn(1, 4, 64, seed=42)
    attend = A.PagedAttention(4, 2, 64)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = attend(q, s.cache, s.batch)
    stream.synchronize()
    close(out, *s.reference(q, 0.125, 0))
    empty = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    s.t_off.zero_()
    assert attend(empty, s.cache, s.batch).shape == (0, 4, 64)
    no_device_error()


# ---- the operators together, in the layers that call them ------------------------------------------------

@pytest.mark.parametrize("hq,hk,d,window", [(4, 2, 64, 40), (2, 1, 256, 0)])
def test_decoder_stack_forward(cuda, hq, hk, d, window):
    """Prompts in chunks, drafted blocks and single tokens of three sequences through two real decoder layers: in
    every layer and step, the queries, the cache and the attention output against the 64-bit forms on the GPU's own
    q|k|v."""
    from helios_b200 import attention as A
    from helios_b200.quantized import synth_normal
    from helios_b200.stack import DecoderStack, StackConfig
    cfg = StackConfig(layers=2, hidden=512, q_out=hq * d, kv_out=hk * d, inter=1024, vocab=2048)
    st = DecoderStack(cfg)
    st.attach_attention(40, 16, head_dim=d, window=window)
    table = torch.randperm(39, generator=torch.Generator().manual_seed(3))[:36].reshape(3, 12).to(torch.int32)
    f = freqs(d, 10000.0)
    have = [0, 0, 0]
    for q_lens in ([70, 9, 0], [33, 1, 150], [1, 1, 1], [5, 5, 5], [1, 0, 1]):
        have = [a + b for a, b in zip(have, q_lens)]
        off = [sum(q_lens[:b]) for b in range(4)]
        n = off[-1]
        batch = A.PagedBatch(torch.tensor(off, dtype=torch.int32, device="cuda"),
                             torch.tensor(have, dtype=torch.int32, device="cuda"), table.cuda(), max_q=max(q_lens))
        h = synth_normal(100 + n, (n, cfg.hidden))
        keep = []
        rows = torch.tensor([o - 1 for o, q in zip(off[1:], q_lens) if q], device="cuda")
        keys, res = st.forward(h, batch, rows=rows, keep=keep)
        no_device_error()
        assert keys.shape == (len(rows),) and torch.isfinite(res).all()
        toks = R.tokens(off, have)
        pos = torch.tensor([t[2] for t in toks])
        page_id, slot = torch.tensor([int(table[b, p // 16]) for _, b, p in toks]), pos % 16
        for L, kept in zip(st.layers, keep):
            qkv = kept["qkv"].cpu()
            q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((hq * d, hk * d, hk * d), 1))
            kc, vc = L["cache"].k.cpu(), L["cache"].v.cpu()
            close(kept["q"], *R.norm_rope(q, pos, f, d, L["q_norm"].cpu(), cfg.eps))
            close(kc[page_id, :, slot], *R.norm_rope(k, pos, f, d, L["k_norm"].cpu(), cfg.eps))
            want = R.norm(v, None, cfg.eps)
            close(vc[page_id, :, slot], want, R.half_step(want) + 2.0 ** -19 * want.abs())
            close(kept["attn"], *R.attention(kept["q"].cpu(), kc, vc, off, have, table.tolist(), d ** -0.5, window))
    st.free()
