"""GPU: attention where the work is many tiles: several of them for every CTA pair, more sequences than a warp has lanes,
contexts up to 16384 keys."""
import pytest
import torch

import attn_ref as R
from test_gpu_attention import Step, close, no_device_error, randn

pytestmark = pytest.mark.gpu


# ---- every key counts once -----------------------------------------------------------------------------

def check_every_key_counts_once(q_lens, kv_lens, hq, hk, d, page, window=0, behind=0):
    """With queries of zero every visible key has the weight 1, in the kernels too: scores, weights and their sums are
    exact. Values that are 1 in the column of their 64-key tile and 0 elsewhere then count the keys of each tile, in
    fp32 exactly; 1 / sum and the product round once each, the output once to bf16. So a tile or a key that is lost,
    counted twice or seen by a row that should not see it shows at any length, where a bound on random values, which
    does not shrink with the context, would hide it."""
    from helios_b200 import attention as A
    s = Step(q_lens, kv_lens, hk, d, page, 17, behind=behind, window=window)
    heads, slots = torch.arange(hk, device="cuda")[:, None], torch.arange(page, device="cuda")
    for b, n in enumerate(kv_lens):
        for p, at in enumerate(s.table[b, : -(-n // page)].tolist()):
            if at >= 0:
                tag = torch.nn.functional.one_hot(((p * page + slots) // 64 + 7 * heads) % d, d).to(torch.bfloat16)
                s.cache.v[at] = torch.where(s.cache.v[at].isnan(), s.cache.v[at], tag)       # unused slots stay NaN
    q = torch.zeros(s.rows, hq, d, dtype=torch.bfloat16, device="cuda")
    out = A.PagedAttention(hq, hk, d)(q, s.cache, s.batch, window=window)
    no_device_error()
    tiles = torch.arange(-(-max(kv_lens) // 64), device="cuda")
    for b, n in enumerate(kv_lens):
        q0, q1 = s.q_offsets[b], s.q_offsets[b + 1]
        if q0 == q1:
            continue
        hi = torch.arange(n - (q1 - q0) + 1, n + 1, device="cuda")[:, None]
        lo = (hi - window).clamp(min=0) if window else torch.zeros_like(hi)
        held = (torch.minimum(hi, 64 * tiles + 64) - torch.maximum(lo, 64 * tiles)).clamp(min=0).double() / (hi - lo)
        for h in range(hk):
            want = torch.zeros(q1 - q0, d, dtype=torch.float64, device="cuda")
            want.index_add_(1, (tiles + 7 * h) % d, held)
            bound = R.half_step(want) + 2.0 ** -22 * want
            err = (out[q0:q1, h * (hq // hk):(h + 1) * (hq // hk)].double() - want[:, None]).abs()
            bad = ~(err <= bound[:, None])
            assert not bad.any(), (b, h, int(bad.sum()), bad.nonzero()[0].tolist())


@pytest.mark.parametrize("q_lens,kv_lens,hq,hk,d,page,window", [
    ([1], [16384], 16, 1, 512, 64, 0),                                     # few rows, every CTA a range
    ([1], [16384], 16, 8, 256, 16, 0),
    ([1] * 5, [16383, 64, 1, 9001, 4097], 16, 8, 256, 32, 0),
    ([1, 1], [12001, 700], 32, 8, 128, 16, 5000),
    ([1], [16384], 12, 4, 64, 128, 0),
    ([8, 8, 3], [2049, 12000, 300], 4, 2, 256, 32, 0),
    ([2, 1], [16000, 4000], 16, 1, 512, 64, 0),
    ([40], [16384], 16, 1, 512, 64, 0),                                    # chunks whose keys are cut into pieces
    ([100, 33], [16384, 9000], 4, 2, 256, 16, 0),
    ([70], [16384], 12, 4, 64, 16, 6000),
    ([1300], [4400], 16, 1, 512, 64, 0),                                   # 2.2 waves of pairs, the last one cut
    ([1300], [4000], 16, 8, 256, 64, 0),                                   # 1.2 waves, cut
    ([1500], [4600], 16, 8, 128, 16, 0),
    ([2900], [2950], 16, 1, 512, 64, 0),                                   # five items a pair
    ([4800], [4800], 16, 8, 256, 64, 0),
    ([4800], [9000], 16, 8, 256, 16, 1024),
    ([2500], [2600], 32, 8, 128, 32, 0),
    ([1700], [1900], 24, 8, 64, 64, 0),
])
def test_every_key_counts_once(cuda, q_lens, kv_lens, hq, hk, d, page, window):
    check_every_key_counts_once(q_lens, kv_lens, hq, hk, d, page, window)


def many_sequences(n, longest, seed):
    g = torch.Generator().manual_seed(seed)
    q = (20 + torch.randint(41, (n,), generator=g)).tolist()
    q[5], q[n // 2] = 0, 1
    return q, [a + b for a, b in zip(q, torch.randint(longest, (n,), generator=g).tolist())]


MANY = [(56, 3000, 4, 2, 256), (40, 3000, 16, 1, 512), (70, 900, 8, 2, 128), (45, 2000, 12, 4, 64), (33, 60, 8, 4, 256)]


@pytest.mark.parametrize("n,longest,hq,hk,d", MANY)
def test_every_key_counts_once_in_many_sequences(cuda, n, longest, hq, hk, d):
    q_lens, kv_lens = many_sequences(n, longest, n)
    check_every_key_counts_once(q_lens, kv_lens, hq, hk, d, 16, behind=2)


# ---- the same sizes with random queries, at sampled rows -----------------------------------------------

def check_sampled_rows(q_lens, kv_lens, hq, hk, d, page, window=0, samples=40):
    from helios_b200 import attention as A
    s = Step(q_lens, kv_lens, hk, d, page, 23, behind=1, window=window)
    q = randn(s.rows, hq, d, seed=24)
    attend = A.PagedAttention(hq, hk, d)
    out = attend(q, s.cache, s.batch, window=window)
    assert torch.equal(attend(q, s.cache, s.batch, window=window)[:-1], out[:-1])
    no_device_error()
    toks = R.tokens(s.q_offsets, kv_lens)
    g = torch.Generator().manual_seed(25)
    at = sorted({0, len(toks) - 1, *torch.randint(len(toks), (samples,), generator=g).tolist()})
    rows, seqs, pos = (list(x) for x in zip(*(toks[i] for i in at)))
    # each sampled row as a sequence of its own that ends with it
    want, bound = R.attention(q.cpu()[rows], s.kc, s.vc, list(range(len(rows) + 1)), [p + 1 for p in pos],
                              [s.table[b].tolist() for b in seqs], d ** -0.5, window)
    close(out[rows], want, bound)


@pytest.mark.parametrize("q_lens,kv_lens,hq,hk,d,page,window", [
    ([1300], [4400], 16, 1, 512, 64, 0),
    ([2900], [2950], 16, 1, 512, 64, 0),
    ([1300], [4000], 16, 8, 256, 64, 0),
    ([4800], [9000], 16, 8, 256, 16, 1024),
    ([2500], [2600], 32, 8, 128, 32, 0),
    ([1700], [1900], 24, 8, 64, 64, 0),
    ([1500, 1, 700, 40, 1], [1500, 5000, 2000, 900, 1], 16, 8, 256, 16, 0),
])
def test_sampled_rows_of_many_tiles(cuda, q_lens, kv_lens, hq, hk, d, page, window):
    check_sampled_rows(q_lens, kv_lens, hq, hk, d, page, window)


@pytest.mark.parametrize("n,longest,hq,hk,d", MANY)
def test_sampled_rows_of_many_sequences(cuda, n, longest, hq, hk, d):
    check_sampled_rows(*many_sequences(n, longest, n), hq, hk, d, 16)
