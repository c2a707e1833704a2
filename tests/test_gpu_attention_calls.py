"""GPU: calls of the attention operators at the edge of what is allowed, and what they refuse."""
import pytest
import torch

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
