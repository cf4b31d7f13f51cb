"""What the operators of long caches refuse, before anything is launched."""
import pytest
import torch

from inference_b200.ops import budget
from inference_b200.ops.runtime import KernelError

B, T, H, KV, D, BS, N = 2, 2, 4, 2, 16, 4, 8


class _NoKernels:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was launched")


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(budget, "kernels", lambda: _NoKernels())
    monkeypatch.setattr(budget, "_place", lambda *a: 0)
    monkeypatch.setattr(budget, "require_cuda", lambda *a: None)


def _args():
    z = torch.zeros
    return {"q": z(T, H, D).bfloat16(), "k": z(20, KV, BS, D).bfloat16(), "v": z(20, KV, BS, D).bfloat16(), "table": z(B, N, dtype=torch.int32),
            "lens": z(B, dtype=torch.int32), "cu": None, "max_q": 1, "w": z(B, KV, N * BS), "pos": z(B, KV, N * BS, dtype=torch.int32), "next": z(B, dtype=torch.int32),
            "codes": z(20, KV, D, dtype=torch.int8), "scales": z(20, KV), "pages": z(T, KV, 3, dtype=torch.int32), "counts": z(T, KV, dtype=torch.int32),
            "keep": 4, "recent": 1, "first": 1, "top": 2, "last": 1, "bs": BS, "splits": None, "out": None}


def _call(name, a):
    step = {"cu_q": a["cu"], "max_q_len": a["max_q"]}
    if name == "summaries":
        return budget.summarize_pages(a["k"], a["table"], a["lens"], budget.PageSummaries(a["codes"], a["scales"]), **step)
    if name == "select":
        return budget.select_pages(a["q"], budget.PageSummaries(a["codes"], a["scales"]), a["table"], a["lens"], block_size=a["bs"], top=a["top"], first=a["first"],
                                   last=a["last"], **step)
    if name == "selected":
        return budget.selected_attention(a["q"], a["k"], a["v"], a["table"], a["lens"], budget.PageSelection(a["pages"], a["counts"]), scale=1.0, num_splits=a["splits"],
                                         out=a["out"], **step)
    if name == "tracked":
        return budget.tracked_attention(a["q"], a["k"], a["v"], a["table"], a["lens"], a["w"], scale=1.0, num_splits=a["splits"], out=a["out"], **step)
    return budget.evict_tokens(a["k"], a["v"], a["table"], a["lens"], a["w"], a["pos"], a["next"], keep=a["keep"], recent=a["recent"], first=a["first"])


ALL = ("summaries", "select", "selected", "tracked", "evict")
CACHED = ("summaries", "selected", "tracked", "evict")
ROWS = ("select", "selected", "tracked")
READ = ("selected", "tracked")

REFUSED = [
    (CACHED, "k", lambda x: x.half()), (CACHED, "k", lambda x: x.transpose(1, 2)), (CACHED, "k", lambda x: x[0]), (CACHED, "k", lambda x: torch.zeros(20, KV, BS, 264).bfloat16()),
    (("selected", "tracked", "evict"), "v", lambda x: x.float()), (("selected", "tracked", "evict"), "v", lambda x: x[:10].contiguous()),
    (("selected", "tracked", "evict"), "v", lambda x: x[:, :1].contiguous()),
    (ALL, "table", lambda x: x.long()), (ALL, "table", lambda x: x[:1]), (ALL, "table", lambda x: x[:, ::2]), (ALL, "table", lambda x: x[:, :0]),
    (ALL, "lens", lambda x: x.long()), (ALL, "lens", lambda x: x[:, None]),
    (("summaries", *ROWS), "cu", lambda x: torch.zeros(B, dtype=torch.int32)), (("summaries", *ROWS), "cu", lambda x: torch.zeros(B + 1)),
    (("summaries", *ROWS), "max_q", lambda x: 0), (ROWS, "max_q", lambda x: 2),
    (ROWS, "q", lambda x: x[:, :3]), (ROWS, "q", lambda x: x[..., :8]), (ROWS, "q", lambda x: x.transpose(0, 2)), (READ, "q", lambda x: x.float()), (("select",), "q", lambda x: x.half()),
    (ROWS, "q", lambda x: torch.zeros(T, 258 * KV, D).bfloat16()),
    (("summaries", "select"), "codes", lambda x: x.to(torch.uint8)), (("summaries",), "codes", lambda x: x[:10]), (("summaries", "select"), "scales", lambda x: x.double()),
    (("summaries", "select"), "scales", lambda x: x[:, :1]), (("summaries", "select"), "codes", lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)),
    (("select",), "top", lambda x: -1), (("select",), "first", lambda x: -1), (("select",), "last", lambda x: 0), (("select",), "bs", lambda x: 0),
    (("select",), "table", lambda x: torch.zeros(B, 60000, dtype=torch.int32)),
    (("selected",), "pages", lambda x: x.long()), (("selected",), "pages", lambda x: x[:1]), (("selected",), "pages", lambda x: x[..., ::2]), (("selected",), "pages", lambda x: x[..., :0]),
    (("selected",), "counts", lambda x: x.float()), (("selected",), "counts", lambda x: x[:, :1]),
    (READ, "splits", lambda x: 0), (READ, "splits", lambda x: 65), (READ, "out", lambda x: torch.zeros(T, H * D)), (READ, "out", lambda x: torch.zeros(T, H * D + 1).bfloat16()),
    (("tracked", "evict"), "w", lambda x: x.double()), (("tracked", "evict"), "w", lambda x: x[..., 1:]), (("tracked", "evict"), "w", lambda x: x[:1].expand(B, -1, -1)),
    (("tracked", "evict"), "w", lambda x: x[:, :1].expand(-1, KV, -1)), (("tracked", "evict"), "w", lambda x: torch.zeros(B, N * BS, KV).transpose(1, 2)),
    (("evict",), "pos", lambda x: x.long()), (("evict",), "pos", lambda x: x[..., 1:]), (("evict",), "pos", lambda x: x[:, :1].expand(-1, KV, -1)),
    (("evict",), "next", lambda x: x.long()), (("evict",), "next", lambda x: x[:1]), (("evict",), "keep", lambda x: 0), (("evict",), "keep", lambda x: 1),
    (("evict",), "recent", lambda x: -1), (("evict",), "first", lambda x: -1),
]


@pytest.mark.parametrize("name,key,change", [(n, k, f) for names, k, f in REFUSED for n in names])
def test_refusals(name, key, change):
    a = _args()
    a[key] = change(a[key])
    with pytest.raises(KernelError):
        _call(name, a)


@pytest.mark.parametrize("name", ALL)
def test_what_is_not_refused_is_launched(name):
    with pytest.raises(AssertionError, match="was launched"):
        _call(name, _args())


def test_tensors_on_the_cpu_are_refused(monkeypatch):
    monkeypatch.undo()
    for name in ALL:
        with pytest.raises(KernelError, match="CUDA tensors"):
            _call(name, _args())


def test_tensors_on_another_device_are_refused(monkeypatch):
    class Elsewhere:
        is_cuda, device = True, "cuda:1"

        def get_device(self):
            return 1

    monkeypatch.undo()
    with pytest.raises(KernelError, match="the current device is cuda:0"):
        budget._place(None, Elsewhere())


def test_rows_that_share_memory():
    x = torch.zeros(3, 4, 10)
    assert not budget._overlaps(x) and not budget._overlaps(x.transpose(0, 1)) and not budget._overlaps(x[:, 1:3, :5])
    assert budget._overlaps(x[:1].expand(3, 4, 10)) and budget._overlaps(torch.as_strided(x, (2, 3, 10), (30, 9, 1))) and budget._overlaps(torch.as_strided(x, (2, 3, 10), (29, 10, 1)))


def test_splits():
    assert budget.budget_splits(8, 100000, True) == 37 and budget.budget_splits(8, 64, True) == 1 and budget.budget_splits(8, 65, False) == 2
    assert budget.budget_splits(8, 8000, False) == 8 and budget.budget_splits(64, 8000, True) == 4 and budget.budget_splits(1, 10 ** 6, True) == 64
    assert budget.budget_splits(400, 10 ** 6, True) == 1 and budget.budget_splits(400, 8192, False) == 7 and budget.budget_splits(10 ** 6, 10 ** 6, False) == 1
    assert budget.budget_splits(64, 4000, True, False) == 18 and budget.budget_splits(8, 100, False, False) == 2 and budget.budget_splits(5000, 4000, False, False) == 1
    assert budget.budget_splits(0, 0, True) == 1 and budget.budget_splits(0, 0, False) == 1


def test_summaries_are_asked_for_before_a_pool_is_used():
    from inference_b200.engine.kv_pool import PagedKvPool, PagedSequence

    pool = PagedKvPool(1, 4, 1, 64, device="cpu")
    PagedSequence(pool).reserve(1)
    with pytest.raises(ValueError):
        pool.with_summaries()
    assert pool.summaries is None
