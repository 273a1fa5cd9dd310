"""Calls of the attention operators that say less than they could."""

import pytest
import torch

import kv_ref
from kv_ref import Pool
from test_gpu_attention import BF16, F16, check, projections

import mlxl3_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new, old", [([1], [40]), ([1, 1, 1], [40, 900, 3]), ([5, 1, 0, 2], [40, 900, 3, 7]), ([2, 0], [9, 30]),
                                      ([70, 33], [0, 500])])
def test_without_max_q_every_row_is_computed(new, old):
    lens = [n + m for n, m in zip(new, old)]
    pool = Pool(90, lens, 2, 64, 16, 8, None)
    cache = pool.cuda(mlxl3_amd)
    told = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    b = mlxl3_amd.KvBatch(told.q_starts, told.kv_lens, told.block_table)
    for rows in (sum(new), sum(new) + 5, sum(new)):  # the same object, with rows behind the last sequence too
        q = torch.randn(rows, 6, 64, generator=torch.Generator().manual_seed(rows)).to(BF16)
        out = torch.full((rows, 6, 64), 7.0, dtype=BF16, device="cuda")
        mlxl3_amd.attention(q.cuda(), cache, b, out=out)
        check(pool, new, q[: sum(new)], out[: sum(new)])
        assert bool((out[sum(new) :] == 7.0).all())


def test_no_tokens_without_max_q():
    pool = Pool(94, [20], 2, 64, 16, 16, F16)
    told = kv_ref.batch(mlxl3_amd, [0], [20], pool.table)
    b = mlxl3_amd.KvBatch(told.q_starts, told.kv_lens, told.block_table)
    none = torch.empty(0, 4, 64, dtype=F16, device="cuda")
    assert mlxl3_amd.attention(none, pool.cuda(mlxl3_amd), b).shape == none.shape


def test_attention_block_without_max_q():
    new, lens, dim, heads, kv_heads = [9, 1, 30], [50, 8, 30], 64, 4, 2
    pool = Pool(91, lens, kv_heads, dim, 16, 16, F16, loud=1.0)
    block = mlxl3_amd.Exl3Attention(*projections(9, 256, heads, kv_heads, dim, 4, 0, False))
    x = torch.randn(sum(new), 256, generator=torch.Generator().manual_seed(3)).half().cuda()
    told = kv_ref.batch(mlxl3_amd, new, lens, pool.table, max_q=sum(new))
    b = mlxl3_amd.KvBatch(told.q_starts, told.kv_lens, told.block_table)
    one, two = pool.cuda(mlxl3_amd), pool.cuda(mlxl3_amd)
    assert torch.equal(block(x, one, b), block(x, two, told))
    for name in "kv":  # bit for bit: slots never written hold NaN
        assert torch.equal(*(getattr(c, name).view(torch.int16) for c in (one, two)))


def test_threads_on_one_stream_share_a_block():
    """Two threads on the default stream, each with its cache: results as one after the other."""
    import threading

    block = mlxl3_amd.Exl3Attention(*projections(10, 256, 4, 2, 64, 4, 0, False))
    sides = []
    for rows in (1, 24):
        pool = Pool(93, [64], 2, 64, 16, 16, F16, poison=False, loud=1.0)
        b = kv_ref.batch(mlxl3_amd, [rows], [64], pool.table)
        x = torch.randn(rows, 256, generator=torch.Generator().manual_seed(rows)).half().cuda()
        sides.append((x, pool.cuda(mlxl3_amd), b))
    want = [block(*s) for s in sides]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            outs = [block(*sides[i]) for _ in range(100)]
            torch.cuda.synchronize()
            failed.extend(f"thread {i}: another result" for y in outs if not torch.equal(y, want[i]))
        except Exception as e:  # told to the main thread
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_arguments_of_the_wrong_kind_are_refused_as_such():
    pool = Pool(92, [20], 2, 64, 16, 16, F16)
    cache, b = pool.cuda(mlxl3_amd), kv_ref.batch(mlxl3_amd, [1], [20], pool.table)
    q = torch.zeros(1, 4, 64, dtype=F16, device="cuda")
    rope = mlxl3_amd.Rope(torch.ones(32, device="cuda"))
    for dtype in (torch.int32, torch.float64):
        with pytest.raises(mlxl3_amd.Exl3Error, match="unsupported rotary output dtype"):
            rope.apply(q, batch=b, dtype=dtype)
    with pytest.raises(mlxl3_amd.Exl3Error, match="out must have q's shape"):
        mlxl3_amd.attention(q, cache, b, out=[1.0])
    with pytest.raises(mlxl3_amd.Exl3Error, match="negative token count"):
        cache.read(b, -1)
    with pytest.raises(mlxl3_amd.Exl3Error, match="attention blocks take f16 or bf16"):
        block = mlxl3_amd.Exl3Attention(*projections(9, 256, 4, 2, 64, 4, 0, False))
        block.workspace_bytes(cache, b, 1, torch.float32)
