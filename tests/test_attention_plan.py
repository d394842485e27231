"""What a plan of attention promises between its build and the calls over it."""
import gc
import weakref

import numpy as np
import pytest
import torch

import cpp_inference_train_engine_amd as mla


class Recorder:
    """Stands in for the library: keeps the arguments of the calls that would launch."""

    def __init__(self):
        self.real, self.calls = mla.lib(), []

    def __getattr__(self, name):
        if name in ("mla_plan_attention", "mla_latent_attention"):
            return lambda *a: self.calls.append((name, a)) or 0
        return getattr(self.real, name)


@pytest.fixture
def recorded(monkeypatch):
    """The wrappers over CPU tensors, every launch recorded in place of made."""
    r = Recorder()
    monkeypatch.setattr(mla.ops, "lib", lambda: r)
    monkeypatch.setattr(mla.ops, "_gpu", lambda: -1)  # where CPU tensors say they are
    monkeypatch.setattr(mla.ops, "stream_handle", lambda stream=None: None)
    return r


def small_batch(B=2, rows=2):
    names = ("cu_seqlens_q", "cu_seqlens_k", "page_table", "slot_mapping", "num_splits", "cu_splits",
             "work_session", "work_split", "work_desc", "work_pages", "info")
    return mla.RaggedBatch(B=B, page_size=64, max_pages=1, num_pool_pages=2, max_work=2, max_rows=rows,
                           **{k: torch.zeros(8, dtype=torch.int32) for k in names})


def small_prefixes():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    return mla.SharedPrefixes(i32(0, 2), i32(70), i32(0, 2), i32(1, 0))


def attend(plan, rows=2):
    q = torch.zeros((rows, 8, 128), dtype=torch.float16)
    mla.latent_attention(plan, torch.zeros((2, 9216), dtype=torch.float16), q,
                         torch.zeros((rows, 8, 16), dtype=torch.float16), 0.1, rope_dim=16, out=q)


def test_a_plan_keeps_the_tensors_that_its_calls_read(recorded):
    """The fields of a batch and of its prefixes may be set anew: calls over an old plan go on with
    what it was made of, which has to stay alive."""
    batch, prefixes = small_batch(), small_prefixes()
    plan = mla.plan_attention(batch, 8, 128, rows=2, max_q_len=1, prefixes=prefixes)
    attend(plan)
    old = [weakref.ref(t) for t in (batch.page_table, prefixes.cu_pages, prefixes.page_ids, plan.words)]
    where = [t().data_ptr() for t in old]
    batch.page_table = torch.ones(8, dtype=torch.int32)
    batch.max_pages, batch.num_pool_pages, batch.page_size = 3, 9, 16
    prefixes.cu_pages = torch.tensor([0, 1], dtype=torch.int32)
    prefixes.page_ids = torch.ones(1, dtype=torch.int32)
    plan.words = None
    gc.collect()
    assert all(t() is not None for t in old), "the plan's calls would read freed memory"
    attend(plan)
    (_, first), (_, second) = recorded.calls[1:]
    for at in (11, 18, 19, 20):  # page table, prefix lists, plan
        assert first[at] == second[at] and first[at] in where
    assert first[5:14] == second[5:14]  # rope, page size, .., max_pages, pool pages
