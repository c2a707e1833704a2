"""GPU: calls of the attention operators at the edge of what is allowed, and what they refuse."""
import pytest
import torch

from test_gpu_attention import Step, no_device_error, randn

pytestmark = pytest.mark.gpu


def bf16(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def one_sequence(tokens, keys, page):
    from helios_b200 import attention as A
    pages = -(-keys // page)
    return A.PagedBatch(int32([0, tokens]), int32([keys]), int32([list(range(pages))]), max_q=tokens)


def test_append_refuses_caches_whose_slots_share_elements(cuda):
    """Keys and values in one tensor, half a page apart, heads or pages over each other: nothing is stored."""
    from helios_b200 import attention as A
    d, page, pages = 64, 16, 3
    rope, batch = A.Rope(d), one_sequence(2, 20, page)
    flat = bf16(8 * pages * page * d, seed=1)
    before = flat.clone()

    def view(start, strides=(2 * page * d, page * d, d, 1), heads=2):
        return flat.as_strided((pages, heads, page, d), strides, start)

    k = bf16(2, 2, d, seed=2)
    far = 4 * pages * page * d
    for kc, vc, word in ((view(0), view(0), "share elements"), (view(0), view(page * d), "share elements"),
                         (view(0), view(8), "share elements"),
                         (view(0, (page * d, page * d, d, 1)), view(far, (page * d, page * d, d, 1)), "must not overlap"),
                         (view(0, (2 * page * d, 8 * d, d, 1)), view(far, (2 * page * d, 8 * d, d, 1)), "must not overlap")):
        with pytest.raises(ValueError, match=word):
            A.kv_append(None, k, k, A.PagedKVCache(kc, vc), batch, rope)
    torch.cuda.synchronize()
    assert torch.equal(flat, before)
    # one tensor for both is read as before
    q = bf16(2, 4, d, seed=3)
    attend = A.PagedAttention(4, 2, d)
    copy = view(0).clone()
    assert torch.equal(attend(q, A.PagedKVCache(view(0), view(0)), batch), attend(q, A.PagedKVCache(copy, copy.clone()), batch))
    # keys and values of a page, of a slot, or of a head in turn qualify
    want = None
    for strides, to_v in (((4 * page * d, page * d, d, 1), 2 * page * d), ((4 * page * d, d, 4 * d, 1), 2 * d),
                          ((4 * page * d, 2 * d, 4 * d, 1), d)):
        flat.zero_()
        cache = A.PagedKVCache(view(0, strides), view(to_v, strides))
        got = A.kv_append(q, k, k, cache, batch, rope)
        stored = got, cache.k.clone(), cache.v.clone()
        assert stored[1].any() and stored[2].any()
        want = want or stored
        assert all(torch.equal(a, b) for a, b in zip(stored, want))


def test_rows_in_the_cache_are_refused(cuda):
    """Inputs and outputs of the append, and the attention's output, that share elements with the pages; between the pages of
    a buffer that holds both they qualify."""
    from helios_b200 import attention as A
    d, page, pages, hk, hq = 64, 16, 3, 2, 4
    block = hk * page * d
    flat = bf16(pages * 4 * block, seed=1)
    shape = pages, hk, page, d
    kc, vc = (flat.as_strided(shape, (4 * block, page * d, d, 1), i * block) for i in range(2))
    cache, batch, rope = A.PagedKVCache(kc, vc), one_sequence(2, 20, page), A.Rope(d)
    q, k, v = bf16(2, hq, d, seed=2), bf16(2, hk, d, seed=3), bf16(2, hk, d, seed=4)
    attend = A.PagedAttention(hq, hk, d)
    before = flat.clone()

    def rows(heads, start, token=None):
        return flat.as_strided((2, heads, d), (token or heads * d, d, 1), start)

    for start in (0, block - hq * d, block, 4 * block + 8, 2 * block - d):       # in k, over its end, in v, later pages
        for bad in ({"q": rows(hq, start)}, {"k": rows(hk, start)}, {"v": rows(hk, start)}, {"q_out": rows(hq, start)}):
            args = {"q": q, "k": k, "v": v, **bad}
            with pytest.raises(ValueError, match="overlaps"):
                A.kv_append(args["q"], args["k"], args["v"], cache, batch, rope, q_out=args.get("q_out"))
        with pytest.raises(ValueError, match="out overlaps the cache"):
            attend(q, cache, batch, out=rows(hq, start))
    torch.cuda.synchronize()
    assert torch.equal(flat, before)
    # tokens of a row each behind a page's values, and heads of queries that are read only anywhere
    free = rows(hq, 2 * block, 4 * block), rows(hk, 3 * block, 4 * block), rows(hk, 3 * block + hk * d, 4 * block)
    for to, x in zip(free, (q, k, v)):
        to.copy_(x)
    want_cache = A.PagedKVCache(kc.clone(), vc.clone())
    want = A.kv_append(q, k, v, want_cache, batch, rope)
    assert torch.equal(A.kv_append(*free, cache, batch, rope, q_out=free[0]), want)
    assert torch.equal(cache.k, want_cache.k) and torch.equal(cache.v, want_cache.v)
    want = attend(want, want_cache, batch)
    assert torch.equal(attend(free[0], cache, batch, out=rows(hq, 2 * block + hq * d, 4 * block)), want)
    inside = rows(hq, 0)
    assert torch.equal(attend(inside, cache, batch), attend(inside.clone(), cache, batch))


def test_outputs_whose_rows_overlap_are_refused(cuda):
    """A token's second head in the place of the next token's first one: two warps would write the row."""
    from helios_b200 import attention as A
    d, hq, hk = 64, 4, 2
    cache = A.PagedKVCache(bf16(3, hk, 16, d, seed=1), bf16(3, hk, 16, d, seed=2))
    batch, rope, attend = one_sequence(3, 40, 16), A.Rope(d), A.PagedAttention(hq, hk, d)
    q, k, v = bf16(3, hq, d, seed=3), bf16(3, hk, d, seed=4), bf16(3, hk, d, seed=5)
    pos = int32([0, 1, 2])
    buf = torch.zeros(64 * d, dtype=torch.bfloat16, device="cuda")
    before = cache.k.clone()

    def rows(heads, token, head):
        return buf.as_strided((3, heads, d), (token, head, 1), 0)

    for token, head in ((d, d), (2 * d, d), (d, 2 * d), (3 * d, d + 8)):
        for call in (lambda: attend(q, cache, batch, out=rows(hq, token, head)),
                     lambda: A.kv_append(q, k, v, cache, batch, rope, q_out=rows(hq, token, head)),
                     lambda: A.qk_norm_rope(q, k, pos, rope, q_out=rows(hq, token, head)),
                     lambda: A.qk_norm_rope(k, q, pos, rope, k_out=rows(hq, token, head))):
            with pytest.raises(ValueError, match="its rows overlap"):
                call()
    torch.cuda.synchronize()
    assert torch.equal(cache.k, before) and not buf.any()
    want = attend(q, cache, batch)
    for token, head in ((hq * d, d), (d, 3 * d), (d, 3 * d + 8), (2 * d, 7 * d)):     # rows of tokens, of heads
        assert torch.equal(attend(q, cache, batch, out=rows(hq, token, head)), want)


@pytest.mark.parametrize("tokens", [1, 3])
def test_outputs_between_other_rows_qualify(cuda, tokens):
    """Rows of different strides whose ends overlap while no element is shared: the keys between two heads of the queries'
    output, a token's outputs behind its inputs in rows of other lengths."""
    from helios_b200 import attention as A
    d, hq, hk = 64, 4, 1
    rope, pos = A.Rope(d), torch.arange(tokens, dtype=torch.int32, device="cuda")
    q, k = bf16(tokens, hq, d, seed=1), bf16(tokens, hk, d, seed=2)
    want = A.qk_norm_rope(q, k, pos, rope)
    buf = torch.zeros(tokens, 16, d, dtype=torch.bfloat16, device="cuda")
    k_in = buf[:, 1:2]
    k_in.copy_(k)
    got = A.qk_norm_rope(q, k_in, pos, rope, q_out=buf[:, 0:8:2], k_out=buf[:, 3:4])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    flat = torch.zeros(128 * d, dtype=torch.bfloat16, device="cuda")          # even places in, odd ones out
    q_in, q_out = flat.as_strided((tokens, hq, d), (16 * d, 2 * d, 1)), flat.as_strided((tokens, hq, d), (32 * d, 4 * d, 1), d)
    q_in.copy_(q)
    assert torch.equal(A.qk_norm_rope(q_in, k, pos, rope, q_out=q_out)[0], want[0])
    with pytest.raises(ValueError, match="overlaps other rows"):
        A.qk_norm_rope(flat.as_strided((tokens, hq, d), (16 * d, 3 * d, 1)), k, pos, rope, q_out=q_out)


def test_fields_assigned_after_the_first_call(cuda):
    """A batch whose max_q and table grow between two steps."""
    from helios_b200 import _lib
    from helios_b200 import attention as A
    cache = A.PagedKVCache(bf16(8, 2, 16, 64, seed=1), bf16(8, 2, 16, 64, seed=2))
    attend, q = A.PagedAttention(4, 2, 64), bf16(5, 4, 64, seed=3)
    batch = one_sequence(1, 16, 16)
    attend(q[:1], cache, batch)
    batch.q_offsets, batch.kv_lens, batch.block_table, batch.max_q = int32([0, 5]), int32([100]), int32([list(range(7))]), 5
    assert torch.equal(attend(q, cache, batch), attend(q, cache, one_sequence(5, 100, 16)))
    assert _lib.device_error() == 0


@pytest.mark.parametrize("hq,hk,d", [(40, 1, 512), (64, 1, 512), (16, 1, 512), (16, 8, 256)])
def test_the_stride_of_a_single_token_is_not_used(cuda, hq, hk, d):
    """More than 32 query heads a key head at head_dim 512 take the chunk kernel with one token too."""
    from helios_b200 import attention as A
    cache = A.PagedKVCache(bf16(5, hk, 16, d, seed=1), bf16(5, hk, 16, d, seed=2))
    batch, attend = one_sequence(1, 70, 16), A.PagedAttention(hq, hk, d)
    q = bf16(1, hq, d, seed=3)
    want = attend(q, cache, batch)
    for stride in (0, 8, 2 ** 41):
        assert torch.equal(attend(q.as_strided((1, hq, d), (stride, d, 1)), cache, batch), want)


def test_two_handles_on_two_streams(cuda):
    """Calls of one token, drafted blocks and chunks of two layers' layouts, each on a stream of its own."""
    from helios_b200 import attention as A
    work = []
    for hq, hk, d, seed in ((16, 8, 256, 41), (16, 1, 512, 43)):
        attend = A.PagedAttention(hq, hk, d)
        for q_lens, kv_lens in (([1], [900]), ([8, 8], [300, 2000]), ([200, 1], [900, 400]), ([700], [1500])):
            s = Step(q_lens, kv_lens, hk, d, 32, seed)
            q = randn(s.rows, hq, d, seed=seed + 1)
            work.append((attend, q, s, attend(q, s.cache, s.batch)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for i in range(4):
            for stream, (attend, q, s, want) in zip(streams, (work[i], work[4 + (i + 1) % 4])):
                with torch.cuda.stream(stream):
                    got.append((attend(q, s.cache, s.batch), want))
    torch.cuda.synchronize()
    no_device_error()
    assert all(torch.equal(a, b) for a, b in got)
