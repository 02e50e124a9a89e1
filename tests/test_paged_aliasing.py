"""What the paged operators hand to their kernels when outputs lie over inputs:
the argument block of each call, taken instead of a launch (CPU). A kernel reads
and writes heads in no order, so a source may share memory with an output only
where it is that output's own and the very same view."""

import itertools

import pytest
import torch

from mtplx_amd import paged_attention, paged_kv_cache, rotary
from mtplx_amd.rotary import apply_rotary, rotary_table

T, H, D = 3, 2, 64


class OnGpu(torch.Tensor):
    """A host tensor that the argument checks take for one on the GPU."""

    is_cuda = property(lambda self: True)


def held(*shape):
    return torch.arange(torch.Size(shape).numel()).reshape(shape).to(torch.bfloat16).as_subclass(OnGpu)


@pytest.fixture
def blocks(monkeypatch):
    """Argument blocks of the calls made, in order."""
    made = []

    def take(name, block, device):
        made.append(block)

    for module in (rotary, paged_kv_cache, paged_attention):
        monkeypatch.setattr(module, "_call", take)
    monkeypatch.setattr(paged_attention, "_workspace", lambda *a: torch.empty(16, dtype=torch.uint8))
    return made


def _elements(ptr, heads, token, head):
    return {ptr + 2 * (t * token + h * head + d) for t, h, d in itertools.product(range(T), range(heads), range(D))}


def check_block(b, in_place=True):
    """No source under another's output; its own output apart or the same rows."""
    src = {"q": (b.q, b.Hq, b.q_token, b.q_head), "k": (b.k, b.Hkv, b.k_token, b.k_head)}
    dst = {"q": (b.q_out, b.Hq, b.qo_token, b.qo_head), "k": (b.k_out, b.Hkv, b.ko_token, b.ko_head)}
    for s, d in itertools.product("qk", "qk"):
        if src[s][0] is None or dst[d][0] is None:
            continue
        if s == d and in_place and src[s] == dst[d]:
            continue
        assert not _elements(*src[s]) & _elements(*dst[d]), f"{s} is read where {d} is written"


def test_a_source_under_another_output_is_copied(blocks):
    t, pos = rotary_table(D, device="cpu"), torch.arange(T)
    x, y, z = held(T, H, D), held(T, H, D), held(T, H, D)
    calls = [(x, x, (x, y)), (x, x, (y, x)), (x, y, (y, x)), (x, y, (z, x)), (x, y, (y, z)), (x, y, (x, y)), (x, x, (y, z))]
    for q, k, out in calls:
        got = apply_rotary(t, q, k, pos, out=out)
        assert got[0] is out[0] and got[1] is out[1]
        check_block(blocks[-1])
    b = blocks[-2]   # (x, y) in place: the caller's own rows
    assert (b.q, b.k) == (b.q_out, b.k_out) == (x.data_ptr(), y.data_ptr())
    # halves that are no whole chunks: not over the own source either
    apply_rotary(rotary_table(24, device="cpu"), x, y, pos, out=(x, y))
    check_block(blocks[-1], in_place=False)


def _parts(fused, *heads):
    """Views [T, h, D] side by side in rows of a fused projection."""
    at, out = 0, []
    for h in heads:
        out.append(fused[:, at * D:(at + h) * D].view(T, h, D))
        at += h
    return out


def test_rotary_in_place_on_a_fused_projection(blocks):
    """Rows that lie side by side share no element: they are read where they are."""
    t, pos = rotary_table(D, device="cpu"), torch.arange(T)
    q, k, _ = _parts(held(T, 8 * D), 4, 2, 2)
    apply_rotary(t, q, k, pos, out=(q, k))
    b = blocks[-1]
    assert (b.q, b.k) == (b.q_out, b.k_out) == (q.data_ptr(), k.data_ptr())
    check_block(b)
    # outputs side by side with sources that are not theirs
    a, x, c, d = _parts(held(T, 8 * D), 2, 2, 2, 2)
    apply_rotary(t, a, x, pos, out=(d, c))
    b = blocks[-1]
    assert (b.q, b.k, b.q_out, b.k_out) == (a.data_ptr(), x.data_ptr(), d.data_ptr(), c.data_ptr())
    apply_rotary(t, a, x, pos, out=(x, c))   # keys under the queries' output
    b = blocks[-1]
    assert b.q == a.data_ptr() and b.k != x.data_ptr()
    check_block(b)


def test_write_and_attention_into_rows_side_by_side(blocks):
    """Queries whose columns only neighbour the output's are read where they are."""
    cache = paged_kv_cache.PagedKVCache(1, 2, D, device="cpu")
    table, start = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q, k, v, out = _parts(held(T, 12 * D), 4, 2, 2, 4)
    for rope in (rotary_table(D, device="cpu"), rotary_table(24, device="cpu")):
        cache.write(k, v, table, start, queries=q, rotary=rope, out=out)
        assert (blocks[-1].q, blocks[-1].q_out) == (q.data_ptr(), out.data_ptr())
    assert paged_attention.paged_sdpa(q, cache, table, start, out=out) is out
    assert (blocks[-1].q, blocks[-1].out) == (q.data_ptr(), out.data_ptr())
    # over the queries themselves: rotated in place, attended from a copy
    cache.write(k, v, table, start, queries=q, rotary=rotary_table(D, device="cpu"), out=q)
    assert blocks[-1].q == blocks[-1].q_out == q.data_ptr()
    cache.write(k, v, table, start, queries=q, rotary=rotary_table(24, device="cpu"), out=q)
    assert blocks[-1].q != blocks[-1].q_out == q.data_ptr()
    paged_attention.paged_sdpa(q, cache, table, start, out=q)
    assert blocks[-1].q != blocks[-1].out == q.data_ptr()


def test_memory_shared_by_two_storages(blocks):
    """The same rows behind another storage (a tensor passed through dlpack)
    are found by their addresses."""
    t, pos = rotary_table(24, device="cpu"), torch.arange(T)
    x = held(T + 1, H, D)
    again = torch.from_dlpack(x.as_subclass(torch.Tensor)[1:]).as_subclass(OnGpu)
    assert again.untyped_storage().data_ptr() != x.untyped_storage().data_ptr() and again.data_ptr() == x[1:].data_ptr()
    apply_rotary(t, x[:T], None, pos, out=(again, None))
    check_block(blocks[-1], in_place=False)
    cache = paged_kv_cache.PagedKVCache(1, H, D, device="cpu")
    table, start = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    paged_attention.paged_sdpa(x[:T], cache, table, start, out=again)
    b = blocks[-1]
    assert not _elements(b.q, H, b.q_token, b.q_head) & _elements(b.out, H, b.out_token, b.out_head)
    with pytest.raises(ValueError):
        cache.write(x[:T], held(T, H, D), table, start, queries=held(T, H, D), rotary=t, out=again)
    # and rows side by side stay apart
    q, k = _parts(held(T, 4 * D), 2, 2)
    k = torch.from_dlpack(k.as_subclass(torch.Tensor)).as_subclass(OnGpu)
    apply_rotary(rotary_table(D, device="cpu"), q, k, pos, out=(q, k))
    b = blocks[-1]
    assert (b.q, b.k) == (b.q_out, b.k_out) == (q.data_ptr(), k.data_ptr())


def test_positions_on_the_host_fit_32_bits(blocks):
    t, x = rotary_table(D, device="cpu"), held(2, H, D)
    for bad in ([0, 2 ** 31], [-2 ** 31 - 1, 0], torch.tensor([2 ** 32, 1]),
                torch.tensor([2 ** 64 - 1, 1], dtype=torch.uint64)):
        with pytest.raises(ValueError):
            apply_rotary(t, x, None, bad)
    assert not blocks
    apply_rotary(t, x, None, [2 ** 31 - 1, -2 ** 31])
    assert len(blocks) == 1


def test_outputs_in_any_order_of_tokens_and_heads(blocks):
    """Rows that do not overlap are written where they lie: heads outside tokens,
    padded rows, a single token or head with any stride."""
    t, pos = rotary_table(D, device="cpu"), torch.arange(T)
    cache = paged_kv_cache.PagedKVCache(1, H, D, device="cpu")
    table, start = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x, kv = held(T, H, D), held(T, H, D)
    outs = [(held(H, T, D).transpose(0, 1), (D, T * D)), (held(H, T, 2 * D)[..., :D].transpose(0, 1), (2 * D, 2 * T * D)),
            (held(T, 3 * H, D)[:, ::3], (3 * H * D, 3 * D)), (held(T, H, D), (H * D, D))]
    for out, strides in outs:
        assert apply_rotary(t, x, None, pos, out=(out, None))[0] is out
        assert (blocks[-1].qo_token, blocks[-1].qo_head) == strides
        assert cache.write(kv, kv, table, start, queries=x, rotary=t, out=out) is out
        assert (blocks[-1].qo_token, blocks[-1].qo_head) == strides
        assert paged_attention.paged_sdpa(x, cache, table, start, out=out) is out
        assert (blocks[-1].out_token, blocks[-1].out_head) == strides
    for n, h in ((1, H), (T, 1), (1, 1)):   # strides of a single token or head are never used
        out = held(T, H, D)[:n, :h].as_strided((n, h, D), (H * D if n > 1 else 3, D if h > 1 else 5, 1))
        y = held(n, h, D)
        assert apply_rotary(t, y, None, pos[:n], out=(out, None))[0] is out
        b = blocks[-1]
        assert b.q_out == out.data_ptr() and b.qo_token % 8 == b.qo_head % 8 == 0 and b.qo_head >= D
    made = len(blocks)
    room = held(4 * T * H * D)
    for strides in ((D, D, 1), (D // 2, T * D, 1), (H * D, D // 2, 1), (D, (T - 1) * D, 1), ((H - 1) * D, D, 1), (0, D, 1),
                    (H * D, 0, 1), (H * D + 4, D, 1), (2 * H * D, 2 * D, 2)):
        with pytest.raises(ValueError):
            apply_rotary(t, x, None, pos, out=(room.as_strided((T, H, D), strides), None))
    with pytest.raises(ValueError):
        apply_rotary(t, x, None, pos, out=(room[1:].as_strided((T, H, D), (H * D, D, 1)), None))
    assert len(blocks) == made


def test_attention_is_refused_where_bits_may_not_depend_on_the_batch(blocks, monkeypatch):
    """A forward inside exact_verify(True) must give a row the same bits in any
    batch; paged_sdpa splits by the lengths of all its requests."""
    from mtplx_amd.attention_context import exact_verify

    monkeypatch.delenv("MTPLX_EXACT_T0_GUARD", raising=False)
    cache = paged_kv_cache.PagedKVCache(1, H, D, device="cpu")
    table, start, x = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), held(T, H, D)
    with exact_verify(True):
        with pytest.raises(RuntimeError, match="exact_verify"):
            paged_attention.paged_sdpa(x, cache, table, start)
        assert not blocks
        cache.write(x, x, table, start)   # (a row's own values alone)
        apply_rotary(rotary_table(D, device="cpu"), x, None, torch.arange(T))
        monkeypatch.setenv("MTPLX_EXACT_T0_GUARD", "0")
        paged_attention.paged_sdpa(x, cache, table, start)
    with exact_verify(False):
        paged_attention.paged_sdpa(x, cache, table, start)
    assert len(blocks) == 4


def test_an_output_that_is_missing(blocks):
    t, pos, x = rotary_table(D, device="cpu"), torch.arange(T), held(T, H, D)
    for out in ((None, x), (held(T, H, D), None)):
        with pytest.raises(TypeError, match="out"):
            apply_rotary(t, x, held(T, H, D), pos, out=out)
    assert not blocks
