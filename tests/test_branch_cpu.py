"""What the operators of drafted trees, page copies and beams refuse, before anything is launched."""
import pytest
import torch

from inference_b200.ops import branch
from inference_b200.ops.runtime import KernelError

B, T, H, KV, D, BS, N = 2, 6, 4, 2, 16, 4, 8


class _NoKernels:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was launched")


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(branch, "kernels", lambda: _NoKernels())
    monkeypatch.setattr(branch, "_place", lambda *a: 0)


def _args():
    z = torch.zeros
    return {"q": z(T, H, D).bfloat16(), "k": z(20, KV, BS, D).bfloat16(), "v": z(20, KV, BS, D).bfloat16(), "table": z(B, N, dtype=torch.int32), "lens": z(B, dtype=torch.int32),
            "cu": None, "max_q": 3, "mask": z(T, 1, dtype=torch.int32), "splits": None, "out": None, "parents": z(T, dtype=torch.int32), "picks": z(T, dtype=torch.int64),
            "tokens": z(T, dtype=torch.int64), "pages": z(3, 2, 20, KV, BS, D), "src": [1, 1, 2], "dst": [3, 4, 5], "logits": z(B * 3, 50), "scores": z(B, 3), "count": 6}


def _call(name, a):
    step = {"cu_q": a["cu"], "max_q_len": a["max_q"]}
    if name == "plan":
        return branch.plan_tree(a["parents"], **step)
    if name == "attention":
        return branch.tree_attention(a["q"], a["k"], a["v"], a["table"], a["lens"], a["mask"], scale=1.0, num_splits=a["splits"], out=a["out"], **step)
    if name == "accept":
        return branch.accept_tree(a["picks"], a["tokens"], a["parents"], a["pages"], a["table"], a["lens"], **step)
    if name == "copy":
        return branch.copy_pages(a["pages"], a["src"], a["dst"])
    return branch.beam_select(a["logits"], a["scores"], count=a["count"])


ALL = ("plan", "attention", "accept", "copy", "beams")
STEP = ("attention", "accept")

REFUSED = [
    (("attention",), "k", lambda x: x.half()), (("attention",), "k", lambda x: x.transpose(1, 2)), (("attention",), "k", lambda x: x[0]),
    (("attention",), "k", lambda x: torch.zeros(20, KV, BS, 264).bfloat16()), (("attention",), "v", lambda x: x.float()), (("attention",), "v", lambda x: x[:10].contiguous()),
    (("attention",), "q", lambda x: x[:, :3]), (("attention",), "q", lambda x: x[..., :8]), (("attention",), "q", lambda x: x.transpose(0, 2)), (("attention",), "q", lambda x: x.float()),
    (("attention",), "q", lambda x: torch.zeros(T, 258 * KV, D).bfloat16()),
    (("attention",), "mask", lambda x: x.long()), (("attention",), "mask", lambda x: x[:1]), (("attention",), "mask", lambda x: x[:, :0]), (("attention",), "mask", lambda x: x[:, 0]),
    (("attention",), "mask", lambda x: torch.zeros(T, 6, dtype=torch.int32)[:, ::2]),
    (("attention",), "splits", lambda x: 0), (("attention",), "splits", lambda x: 65),
    (("attention",), "out", lambda x: torch.zeros(T, H * D)), (("attention",), "out", lambda x: torch.zeros(T, H * D + 1).bfloat16()),
    (("attention",), "out", lambda x: torch.zeros(1, H * D).bfloat16().expand(T, -1)),
    (STEP, "table", lambda x: x.long()), (STEP, "table", lambda x: x[:1]), (STEP, "table", lambda x: x[:, ::2]), (STEP, "table", lambda x: x[:, :0]),
    (STEP, "lens", lambda x: x.long()), (STEP, "lens", lambda x: x[:, None]),
    (STEP, "cu", lambda x: torch.zeros(B, dtype=torch.int32)), ((*STEP, "plan"), "cu", lambda x: torch.zeros(B + 1)),
    ((*STEP, "plan"), "max_q", lambda x: 0), ((*STEP, "plan"), "max_q", lambda x: 4), ((*STEP, "plan"), "max_q", lambda x: 2 ** 31),
    (("plan", "accept"), "parents", lambda x: x.long()), (("plan", "accept"), "parents", lambda x: x[:, None]), (("accept",), "parents", lambda x: x[:3]),
    (("plan", "accept"), "parents", lambda x: torch.zeros(2 * T, dtype=torch.int32)[::2]),
    (("accept",), "picks", lambda x: x.int()), (("accept",), "picks", lambda x: x[:3]), (("accept",), "tokens", lambda x: x.int()), (("accept",), "tokens", lambda x: x[:3]),
    (("accept",), "tokens", lambda x: torch.zeros(2 * T, dtype=torch.int64)[::2]),
    (("accept", "copy"), "pages", lambda x: x[0]), (("accept", "copy"), "pages", lambda x: x.transpose(0, 1)), (("accept", "copy"), "pages", lambda x: [x[0, 0], x[0, 0, :5]]),
    (("accept", "copy"), "pages", lambda x: [x[0, 0].transpose(1, 2)]), (("accept",), "pages", lambda x: [x[0]]), (("accept",), "pages", lambda x: [x[0, 0], x[0, 0, :, :, :2].contiguous()]),
    (("accept",), "pages", lambda x: [x[0, 0], x[0, 0]]),
    (("copy",), "src", lambda x: [1, 1]), (("copy",), "src", lambda x: [1, 1, 20]), (("copy",), "src", lambda x: [1, 1, -1]), (("copy",), "src", lambda x: [1, 3, 2]),
    (("copy",), "dst", lambda x: [3, 4, 3]), (("copy",), "dst", lambda x: [3, 4, 20]), (("copy",), "dst", lambda x: [3, 4, -1]), (("copy",), "dst", lambda x: torch.zeros(3, dtype=torch.int32)),
    (("copy",), "src", lambda x: torch.zeros(3, dtype=torch.int32)),
    (("beams",), "logits", lambda x: x.half()), (("beams",), "logits", lambda x: x[:5]), (("beams",), "logits", lambda x: x[:, ::2]), (("beams",), "logits", lambda x: x[:, :0]),
    (("beams",), "logits", lambda x: x[None]), (("beams",), "scores", lambda x: x.double()), (("beams",), "scores", lambda x: x.view(-1)), (("beams",), "scores", lambda x: x.view(1, 6).T[:, :1].expand(-1, 1)[:4]),
    (("beams",), "count", lambda x: 0), (("beams",), "count", lambda x: 129),
]


@pytest.mark.parametrize("name,key,change", [(n, k, f) for names, k, f in REFUSED for n in names])
def test_refusals(name, key, change):
    a = _args()
    a[key] = change(a[key])
    with pytest.raises(KernelError):
        _call(name, a)


@pytest.mark.parametrize("name", ALL)
def test_what_is_not_refused_reaches_the_library(name):
    with pytest.raises(AssertionError, match="was launched"):
        _call(name, _args())


def test_lists_of_device_pages_are_int32():
    a = _args()
    a["src"], a["dst"] = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(KernelError):
        _call("copy", a)


def test_more_beams_than_the_kernel_takes():
    with pytest.raises(KernelError):
        branch.beam_select(torch.zeros(257, 5), torch.zeros(1, 257), count=3)
