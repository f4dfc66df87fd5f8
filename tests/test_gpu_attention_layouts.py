"""Layouts and sizes of the attention that its kernels treat on their own: caches with
the heads outside, keys shared by a batch, many sequences and many pieces, element
offsets past 2^31, lengths that change under a captured graph. Tolerances as in
test_gpu_attention."""
import pytest
import torch

from lynnreal_omni_amd import _lib
from lynnreal_omni_amd import attention as A
from test_gpu_attention import check, formula, mask, tensors

pytestmark = pytest.mark.gpu

LENGTHS = 2     # lr_attention_splits' kind of a batch with key lengths


def pieces(n, rows, size, heads, kv_heads):
    return _lib.load().lr_attention_splits(n, rows, size, LENGTHS, heads, kv_heads)


@pytest.mark.parametrize("new", [1, 2, 50])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_caches_with_the_heads_outside(new, dtype, dim):
    """[batch, heads, tokens, dim] seen through a transpose: taken as it is, the same bits."""
    lengths, size = [700, 0, 33, 512], 700
    g = torch.Generator().manual_seed(new)
    q = torch.randn(4, new, 6, dim, generator=g).to(dtype).cuda()
    k, v = (torch.randn(4, 2, size, dim, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    assert A._rows(k).data_ptr() == k.data_ptr() and not k.is_contiguous()
    given = torch.tensor(lengths, device="cuda")
    for causal in (False, True):
        got = A.attention(q, k, v, causal=causal, key_lengths=given)
        for i, n in enumerate(lengths):
            check(got[i], *formula(q[i], k[i, :n], v[i, :n], dim ** -0.5, mask(new, n, causal)))
        assert torch.equal(got, A.attention(q, k.contiguous(), v.contiguous(), causal=causal, key_lengths=given))
        whole = A.attention(q, k, v, causal=causal)
        assert torch.equal(whole, A.attention(q, k.contiguous(), v.contiguous(), causal=causal))
    packed = A.attention_packed(q[0], k[0], v[0], torch.tensor([0, new], device="cuda"),
                                torch.tensor([0, size], device="cuda"))
    check(packed, *formula(q[0], k[0], v[0], dim ** -0.5, mask(new, size, False)))


@pytest.mark.parametrize("new", [1, 70])
def test_keys_shared_by_a_batch(new):
    """Keys and values expanded over the batch (stride 0), and a query expanded over its tokens."""
    batch, size, dim = 5, 900, 64
    q, k, v = tensors(batch * new, size, 4, 2, dim, torch.bfloat16, new)
    q = q.view(batch, new, 4, dim)
    ke, ve = (t[None].expand(batch, -1, -1, -1) for t in (k, v))
    given = torch.tensor([900, 1, 0, 899, 64], device="cuda", dtype=torch.int32)
    for lengths in (None, given):
        got = A.attention(q, ke, ve, key_lengths=lengths)
        for i in range(batch):
            n = size if lengths is None else lengths[i].item()
            check(got[i], *formula(q[i], k[:n], v[:n], dim ** -0.5, mask(new, n, False)))
    same = q[:1, :1].expand(batch, new, -1, -1)
    assert torch.equal(A.attention(same, ke, ve), A.attention(same.contiguous(), ke.contiguous(), ve.contiguous()))


@pytest.mark.parametrize("new,heads", [(1, 4), (3, 2)])
@pytest.mark.parametrize("batch", [64, 65, 130, 200])
def test_more_sequences_than_a_wave_has_lanes(batch, new, heads):
    """The list of pieces over groups of 64 sequences, empty ones at their ends."""
    size, dim = 700, 64
    assert pieces(batch, new, size, heads, 1) >= 2 * batch
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 200, (batch,), generator=g)
    lengths[[0, 63, batch - 1]] = 0
    lengths[[5, 62, batch - 2]] = size
    q = torch.randn(batch, new, heads, dim, generator=g).half().cuda()
    k, v = (torch.randn(batch, size, 1, dim, generator=g).half().cuda() for _ in range(2))
    got = A.attention(q, k, v, causal=True, key_lengths=lengths.cuda())
    for i, n in enumerate(lengths.tolist()):
        check(got[i], *formula(q[i], k[i, :n], v[i, :n], dim ** -0.5, mask(new, n, True)))


@pytest.mark.parametrize("heads", [1, 4, 160])
def test_most_pieces_of_a_sequence(heads):
    """256 splits of one sequence, and lists with more places than that; 160 query heads
    of one key head take more than a tile for a single token."""
    keys, dim = 40000, 32
    q, k, v = tensors(1, keys, heads, 1, dim, torch.bfloat16, heads)
    want = formula(q, k, v, dim ** -0.5, mask(1, keys, False))
    if heads == 4:
        assert _lib.load().lr_attention_splits(1, 1, keys, 0, heads, 1) == 256
        assert pieces(2, 1, keys, heads, 1) > 256
    check(A.attention(q[None], k[None], v[None])[0], *want)
    for lengths in ([keys], [keys, 17], [0, keys, 64, 0]):
        n = len(lengths)
        got = A.attention(q.expand(n, 1, -1, -1), k.expand(n, -1, -1, -1), v.expand(n, -1, -1, -1),
                          key_lengths=torch.tensor(lengths, device="cuda"))
        for i, length in enumerate(lengths):
            check(got[i], *(want if length == keys else
                            formula(q, k[:length], v[:length], dim ** -0.5, mask(1, length, False))))


def test_sequences_past_2_31_elements():
    """The last of nine caches begins at element 2^31."""
    size, heads, dim, n = 1 << 18, 8, 128, 300
    k, v = (torch.zeros(9, size, heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    assert 8 * k.stride(0) == 1 << 31
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in (k, v):
        t[:, :n] = torch.randn(9, n, heads, dim, device="cuda", generator=g).bfloat16()
    q = torch.randn(9, 2, heads, dim, device="cuda", generator=g).bfloat16()
    got = A.attention(q, k, v, key_lengths=torch.full((9,), n, device="cuda"))
    for i in (0, 8):
        check(got[i], *formula(q[i], k[i, :n], v[i, :n], dim ** -0.5, mask(2, n, False)))
    whole = A.attention(q, k[:, :n], v[:, :n])
    for i in (0, 8):
        check(whole[i], *formula(q[i], k[i, :n], v[i, :n], dim ** -0.5, mask(2, n, False)))


def test_tokens_past_2_31_elements():
    """Tokens 2^22 elements apart: those from 512 on lie past 2^31, in the keys, the
    values and the queries, in one sequence and as the first of a packed one."""
    tokens, apart, dim = 600, 1 << 22, 64
    rows = torch.empty(tokens, apart, device="cuda", dtype=torch.bfloat16)
    rows[:, :3 * dim] = torch.randn(tokens, 3 * dim, device="cuda",
                                    generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    q, k, v = (rows[:, i * dim:(i + 1) * dim].unflatten(1, (1, dim)) for i in range(3))
    assert k.stride(0) * 512 == 1 << 31 and A._rows(k).data_ptr() == k.data_ptr()
    for causal in (False, True):
        got = A.attention(q[None], k[None], v[None], causal=causal)[0]
        check(got, *formula(q, k, v, dim ** -0.5, mask(tokens, tokens, causal)))
    one = A.attention(q[None, -1:], k[None], v[None])[0]
    check(one, *formula(q[-1:], k, v, dim ** -0.5, mask(1, tokens, False)))
    cu = [0, 7, 520, 600]
    packed = A.attention_packed(q, k, v, torch.tensor(cu, device="cuda"))
    for a, b in zip(cu, cu[1:]):
        check(packed[a:b], *formula(q[a:b], k[a:b], v[a:b], dim ** -0.5, mask(b - a, b - a, False)))


def test_outputs_past_2_31_elements():
    """131200 tokens of 128 heads of 128: the last outputs lie past 2^31 elements. One
    query of all tokens (stride 0), so that all rows are one."""
    tokens, heads, dim = 131200, 128, 128
    q, k, v = tensors(1, 40, heads, heads, dim, torch.bfloat16, 5)
    out = A.attention(q.expand(tokens, -1, -1)[None], k[None], v[None])[0]
    assert out.numel() > 1 << 31
    check(out[:1], *formula(q, k, v, dim ** -0.5, mask(1, 40, False)))
    assert all((part == out[:1]).all() for part in out.split(16384))


@pytest.mark.parametrize("size", [64, 3000])
def test_lengths_that_change_under_a_graph(size):
    """A captured step of a batch of caches: the lengths, the new keys and the query are
    those of each replay, also where a cache empties or fills up."""
    batch, heads, kv_heads, dim = 4, 8, 2, 64
    g = torch.Generator().manual_seed(size)
    q = torch.randn(batch, 1, heads, dim, generator=g).bfloat16().cuda()
    k, v = (torch.randn(batch, size, kv_heads, dim, generator=g).bfloat16().cuda() for _ in range(2))
    lengths = torch.full((batch,), size // 2, device="cuda", dtype=torch.int32)
    A.attention(q, k, v, key_lengths=lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.attention(q, k, v, key_lengths=lengths)
    for step in ([size, 1, 0, 33], [0, 0, 0, 0], [size] * 4, [2, size - 1, 64, 0]):
        lengths.copy_(torch.tensor(step))
        q.copy_(torch.randn(q.shape, generator=g))
        k[:, :2] = torch.randn(batch, 2, kv_heads, dim, generator=g).bfloat16().cuda()
        graph.replay()
        want = A.attention(q, k, v, key_lengths=lengths)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for i, n in enumerate(step):
            check(out[i], *formula(q[i], k[i, :n], v[i, :n], dim ** -0.5, mask(1, n, False)))
