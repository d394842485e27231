"""Attention over the paged key-value cache in batches that fill the GPU: blocks of many rows that are
left whole over long contexts, more blocks than workgroups with and without cuts, several ranges for
each workgroup, and a step of decode rows, drafts and chunks that runs both kernels at length."""
import pytest
import torch

from kv_reference import Batch, TYPE, near, say

F16, BF16 = 0, 1


def hold(gpu, c, window=None, sinks=0):
    """Rows and lse as the formula gives them; returns {jobs, 0, of few rows, of many, partial rows}."""
    batch, cache, q = c.device(gpu)
    plan = gpu.plan_kv_attention(batch, cache, c.H, rows=c.rows, max_q_len=max(c.q_len), window=window,
                                 sinks=sinks)
    want, want_lse, off, off_lse = c.expect(window, sinks)
    info = plan.read_info()
    lse = torch.zeros((c.rows, c.H), device="cuda")
    near(gpu.kv_attention(plan, cache, 0, q, c.scale, lse=lse), want, off, "out")
    near(lse, want_lse, off_lse, "lse")
    return info[:5]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,DV,page,rows", [(128, 128, 64, 4100), (64, 64, 48, 5000), (192, 128, 16, 4100),
                                            (256, 256, 32, 2100)])
def test_whole_blocks_over_long_contexts(gpu, D, DV, page, rows, dtype):
    """A prompt of 16 heads on one: blocks of 8 tokens, more than workgroups, the last over all keys."""
    say(f"whole blocks {D} {rows} {dtype}")
    c = Batch(16, 1, D, DV, page, dtype, [(50, rows)], seed=D)
    blocks = -(-rows * 16 // 128)
    assert hold(gpu, c) == [blocks, 0, 0, blocks, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (3000, 70)])
def test_more_blocks_than_workgroups_and_one_long_session(gpu, window, sinks):
    say(f"one long session {window}")
    # many rows: 520 sessions of a block each, 13 blocks of 100 rows on 6,000 tokens
    c = Batch(16, 1, 64, 64, 64, BF16, [(i % 50, 8) for i in range(520)] + [(6000, 100)], seed=1)
    info = hold(gpu, c, window, sinks)
    assert info[3] > 520 + 13 and info[4] > 0
    # few rows: a hundred short sessions of 16 heads, one of 6,400 tokens
    c = Batch(16, 16, 64, 64, 64, F16, [(i % 50, 1) for i in range(100)] + [(6400, 1)], seed=2)
    info = hold(gpu, c, window, sinks)
    assert info[2] > 101 and info[4] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_several_ranges_for_each_workgroup(gpu, dtype):
    """Long uneven sessions of 64 heads: the GPU holds 24 workgroups of each."""
    say(f"several ranges {dtype}")
    c = Batch(64, 64, 16, 16, 64, dtype, [(1500 + 33 * i, 1) for i in range(19)] + [(6400, 1)], seed=3)
    info = hold(gpu, c)
    assert info[2] > 24 and info[4] == info[2]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 4)])
def test_a_step_of_decode_rows_drafts_and_chunks(gpu, window, sinks):
    say(f"mixed step {window}")
    sessions = [(300 + 97 * i, 1) for i in range(40)] + [(200 + 150 * i, 5) for i in range(8)] + \
               [(0, 700), (1500, 512), (3000, 512), (64, 130)]
    c = Batch(32, 8, 128, 128, 64, BF16, sessions, seed=4)
    info = hold(gpu, c, window, sinks)
    assert info[2] > 0 and info[3] > 0
