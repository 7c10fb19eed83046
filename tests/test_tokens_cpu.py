"""CPU: the token operators' entry points refuse what they can not compute before anything is launched, size their
workspaces without overflow, and the Python layer has no CPU path."""
import ctypes as C

import pytest
import torch

from diffusion_model_ligandmol_generation_amd import _lib
from diffusion_model_ligandmol_generation_amd import tokens as tk

ARG, WS = 1, 2
P = 0x1000   # never dereferenced: every call below is refused on the host


def rows(**kw):
    a = _lib.TokenArgs(P, P, 119, 10, 119, _lib.DTYPE_F32, 8, 1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(vocab=0), dict(vocab=-3), dict(row_stride=118), dict(row_stride=0), dict(n_tokens=-1),
                                dict(n_tokens=1 << 31), dict(dtype=3), dict(dtype=-1), dict(token_bytes=2),
                                dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                                dict(temperature=float("inf")), dict(temperature=1e-21), dict(temperature=1e21), dict(logits=None),
                                dict(tokens=None)])
def test_token_rows_are_checked(lib, kw):
    a = rows(**kw)
    assert lib.ligdiff_token_logprob(C.byref(a), P, P, None) == ARG
    assert lib.ligdiff_token_logprob_grad(C.byref(a), P, P, None, 10, 1.0, None, P, 119, None) == ARG
    q = preference()
    assert lib.ligdiff_preference_loss(C.byref(a), C.byref(q), None) == ARG
    q = policy()
    assert lib.ligdiff_policy_loss(C.byref(a), C.byref(q), None) == ARG


def test_logprob_outputs_are_checked(lib):
    a = rows()
    assert lib.ligdiff_token_logprob(C.byref(a), None, P, None) == ARG
    assert lib.ligdiff_token_logprob(None, P, P, None) == ARG
    for args in ((None, P, None, 10, 1.0, None, P, 119), (P, None, None, 10, 1.0, None, P, 119), (P, P, None, 10, 1.0, None, None, 119),
                 (P, P, None, 10, 1.0, None, P, 118), (P, P, None, 9, 1.0, None, P, 119), (P, P, P, 0, 1.0, None, P, 119)):
        assert lib.ligdiff_token_logprob_grad(C.byref(a), *args, None) == ARG


def preference(**kw):
    q = _lib.PreferenceArgs(P, P, 2, 0, 0, 0.1, 0.0, 0.0, 1.0, P, P, P, P, P, P, P, 119, P, 1 << 30)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize("kw", [dict(seq_ptr=None), dict(n_pairs=0), dict(n_pairs=-1), dict(n_pairs=0x40000000), dict(kind=2),
                                dict(beta=0.0), dict(beta=float("nan")), dict(beta=float("inf")), dict(label_smoothing=0.5),
                                dict(label_smoothing=-0.1), dict(label_smoothing=float("nan")), dict(denominator=float("nan")),
                                dict(grad_scale=float("nan")), dict(loss=None), dict(log_ratio=None), dict(margin=None),
                                dict(slope=None), dict(stats=None), dict(row_seq=None), dict(d_stride=118), dict(workspace=None)])
def test_preference_is_checked(lib, kw):
    a, q = rows(), preference(**kw)
    assert lib.ligdiff_preference_loss(C.byref(a), C.byref(q), None) == ARG


def policy(**kw):
    q = _lib.PolicyArgs(P, P, P, P, 2, 0, 0, 0.2, 0.2, 0.1, 0.0, 1.0, P, P, P, P, P, 119, P, 1 << 30)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize("kw", [dict(n_seq=0), dict(n_seq=-1), dict(seq_ptr=None), dict(advantage=None), dict(aggregate=2),
                                dict(clip_low=-0.1), dict(clip_low=1.5), dict(clip_low=float("nan")), dict(clip_high=-0.1),
                                dict(clip_high=float("inf")), dict(kl_coef=-1.0), dict(kl_coef=float("nan")), dict(result=None),
                                dict(d_stride=100), dict(workspace=None), dict(grad_scale=float("nan")),
                                dict(denominator=float("nan"))])
def test_policy_is_checked(lib, kw):
    a, q = rows(), policy(**kw)
    assert lib.ligdiff_policy_loss(C.byref(a), C.byref(q), None) == ARG


def test_small_workspaces_are_refused(lib):
    a = rows(n_tokens=5000)
    need = lib.ligdiff_preference_workspace_bytes(5000, 2)
    q = preference(workspace_bytes=need - 1)
    assert lib.ligdiff_preference_loss(C.byref(a), C.byref(q), None) == WS
    for mean in (0, 1):
        need = lib.ligdiff_policy_workspace_bytes(5000, 2, mean)
        q = policy(workspace_bytes=need - 1, aggregate=mean)
        assert lib.ligdiff_policy_loss(C.byref(a), C.byref(q), None) == WS
    need = lib.ligdiff_embed_grad_workspace_bytes(5000, 119, 256)
    assert lib.ligdiff_embed_grad(P, 0, 256, P, 8, 5000, 119, 256, 1.0, P, 0, 256, 0, P, need - 1, None) == WS


def test_workspace_sizes(lib):
    f = lib.ligdiff_embed_grad_workspace_bytes
    assert f(-1, 119, 256) == 0 and f(10, 0, 256) == 0 and f(10, 119, 0) == 0 and f(1 << 31, 119, 256) == 0 and f(10, 1 << 31, 1) == 0
    assert f(0, 119, 256) > 0 and f(29696, 119, 256) < f(59392, 119, 256)
    # two sorted copies of the positions, and partial rows of at most an eighth of fp32 rows
    big = f(1 << 30, 1 << 20, 4096)
    assert 4 * 4 * (1 << 30) < big < 4 * 4 * (1 << 30) + (1 << 30) * 4096 * 4 // 8 + (1 << 24)
    g = lib.ligdiff_preference_workspace_bytes
    assert g(-1, 1) == 0 and g(1, 0) == 0 and g(1 << 31, 1) == 0 and g(0, 1) > 0 and g(2 ** 31 - 1, 2 ** 20) > 4 * (2 ** 31 - 1)
    h = lib.ligdiff_policy_workspace_bytes
    assert h(-1, 1, 0) == 0 and h(1, 0, 0) == 0 and h(0, 1, 1) > 0 and h(2 ** 31 - 1, 2 ** 31 - 1, 1) > 8 * (2 ** 31 - 1)


@pytest.mark.parametrize("args", [
    (P, 3, 119, 256, 256, P, 8, 10, 1.0, P, 256), (P, 0, 0, 256, 256, P, 8, 10, 1.0, P, 256), (P, 0, 119, 0, 256, P, 8, 10, 1.0, P, 256),
    (P, 0, 119, 256, 255, P, 8, 10, 1.0, P, 256), (P, 0, 119, 256, 256, P, 3, 10, 1.0, P, 256), (P, 0, 119, 256, 256, P, 8, -1, 1.0, P, 256),
    (P, 0, 119, 256, 256, P, 8, 10, 1.0, P, 255), (None, 0, 119, 256, 256, P, 8, 10, 1.0, P, 256),
    (P, 0, 119, 256, 256, None, 8, 10, 1.0, P, 256), (P, 0, 119, 256, 256, P, 8, 10, 1.0, None, 256),
    (P, 0, 1 << 31, 256, 256, P, 8, 10, 1.0, P, 256)])
def test_embed_is_checked(lib, args):
    assert lib.ligdiff_embed(*args, None) == ARG


@pytest.mark.parametrize("args", [
    (P, 1, 256, P, 8, 10, 119, 256, 1.0, P, 2, 256, 0, P), (P, 0, 255, P, 8, 10, 119, 256, 1.0, P, 0, 256, 0, P),
    (P, 0, 256, P, 8, 10, 119, 256, 1.0, P, 0, 255, 0, P), (P, 0, 256, P, 8, 10, 119, 256, 1.0, None, 0, 256, 0, P),
    (None, 0, 256, P, 8, 10, 119, 256, 1.0, P, 0, 256, 0, P), (P, 0, 256, None, 8, 10, 119, 256, 1.0, P, 0, 256, 0, P),
    (P, 0, 256, P, 8, 10, 119, 256, 1.0, P, 0, 256, 0, None), (P, 0, 256, P, 5, 10, 119, 256, 1.0, P, 0, 256, 0, P),
    (P, 0, 256, P, 8, 1 << 31, 119, 256, 1.0, P, 0, 256, 0, P), (P, 0, 256, P, 8, 10, 0, 256, 1.0, P, 0, 256, 0, P)])
def test_embed_grad_is_checked(lib, args):
    assert lib.ligdiff_embed_grad(*args, 1 << 30, None) == ARG


def test_no_cpu_path():
    x, ids, ptr = torch.zeros(4, 119), torch.zeros(4, dtype=torch.int64), torch.tensor([0, 2, 4], dtype=torch.int32)
    for call in (lambda: tk.embed_tokens(ids, x), lambda: tk.embed_tokens_grad(x, ids, 9), lambda: tk.token_logprobs(x, ids),
                 lambda: tk.preference_loss(x, ids, ptr), lambda: tk.policy_loss(x, ids, ptr, torch.zeros(2)),
                 lambda: tk.token_logprobs(x.requires_grad_(), ids)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def _count_worker(rank, world, port, q):
    import os
    import torch.distributed as dist
    from types import SimpleNamespace
    from diffusion_model_ligandmol_generation_amd.train import ResearchAccurateTrainer
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    me = SimpleNamespace(group=dist.group.WORLD, count_group=dist.group.WORLD)
    q.put(ResearchAccurateTrainer._sum_over_ranks(me, 10 ** 9 + rank, 3 - rank))
    dist.destroy_process_group()


def test_counts_over_ranks():
    """The denominators of the fine-tuning steps are the counts of all ranks (two gloo processes)."""
    import socket
    from types import SimpleNamespace
    import torch.multiprocessing as mp
    from diffusion_model_ligandmol_generation_amd.train import ResearchAccurateTrainer
    assert ResearchAccurateTrainer._sum_over_ranks(SimpleNamespace(group=None), 7) == (7,)
    with socket.socket() as sock:
        sock.bind(("127.0.0.1", 0))
        port = sock.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_count_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(60)
    assert got == [(2 * 10 ** 9 + 1, 5)] * 2 and all(p.exitcode == 0 for p in procs)
