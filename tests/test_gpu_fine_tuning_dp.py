"""GPU: fine-tuning steps of two data-parallel ranks (gloo, both on cuda:0) against one process with the whole batch: the same
gradients, dropout masks among what is the same, and shares of the loss that add up.  Gradients are held to the 1e-4 (2-norm
of a parameter's difference over that of its gradient) of the suite's other forms of the network."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_gpu_atom_types import Bag, model_of, trainer_of
from test_gpu_fine_tuning import dropout_model

pytestmark = pytest.mark.gpu

SIZES = [9, 14, 3, 20, 29, 7, 11, 26]      # the first four on rank 0, the others on rank 1
KEY = 1234567


def molecules():
    from oracle import template_connectivity
    g = torch.Generator().manual_seed(5)
    out = []
    for n in SIZES:
        types = torch.tensor([1, 6, 7, 8, 9])[torch.multinomial(torch.tensor([.3, .5, .09, .09, .02]), n, True, generator=g)]
        types[torch.rand(n, generator=g) < 0.15] = -1
        out.append(dict(x=torch.randn(n, 119, generator=g), pos=1.5 * torch.randn(n, 3, generator=g), types=types,
                        edges=torch.tensor(template_connectivity(n)[0], dtype=torch.int64).reshape(-1, 2).t(),
                        u=torch.rand(1, generator=g), noise=torch.randn(n, 3, generator=g), adv=torch.randn(1, generator=g),
                        old=-4.8 + 0.2 * torch.randn(n, generator=g)))
    return out


def batch_of(mols):
    b, off, edges = Bag(), 0, []
    for m in mols:
        edges.append(m["edges"] + off)
        off += len(m["types"])
    cat = lambda k: torch.cat([m[k] for m in mols]).cuda()      # noqa: E731
    b.x, b.pos, b.atom_types, b.edge_index = cat("x"), cat("pos"), cat("types"), torch.cat(edges, 1).cuda()
    b.batch = torch.repeat_interleave(torch.arange(len(mols)), torch.tensor([len(m["types"]) for m in mols])).cuda()
    return b, dict(u=cat("u"), noise=cat("noise"), dropout_seed=KEY), cat("adv"), cat("old")


def pairs_of(mols):
    """Preferred ones first: mols are (preferred, other) in turn."""
    return mols[0::2] + mols[1::2]


def all_steps(group, mols):
    """Loss, log-probabilities and gradients of every kind of step on these molecules."""
    out = {}

    def run(name, model, step):
        tr = trainer_of(model, process_group=group)
        got = {}
        tr.optimizer.clip_and_step = lambda *a, **k: got.update({n: p.grad.cpu() for n, p in tr.model.named_parameters() if p.grad is not None})
        r = step(tr)
        out[name] = (float(r.loss), got)

    b, draws, adv, old = batch_of(mols)
    for aggregate in ("token", "sequence"):
        run("policy " + aggregate, dropout_model(), lambda tr: tr.policy_step(b, draws, adv, old, old, kl_coef=0.1, aggregate=aggregate))
        scored = []
        run("scored " + aggregate, dropout_model(),     # masks fixed by the scoring call
            lambda tr: tr.policy_step(b, scored.append(tr.atom_type_logprobs(b, draws)) or scored[0][1], adv, scored[0][0], kl_coef=0.0,
                                      aggregate=aggregate))
    bp, dp, _, old_p = batch_of(pairs_of(mols))
    run("preference", model_of(), lambda tr: tr.preference_step(bp, dp, old_p, beta=0.3, label_smoothing=0.1))
    b.atom_types = torch.full_like(b.atom_types, -1)
    run("nothing", model_of(), lambda tr: tr.policy_step(b, draws, adv, old))
    return out


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)
    out = all_steps(dist.group.WORLD, molecules()[rank * 4:rank * 4 + 4])
    q.put((rank, {k: (loss, {n: t.numpy() for n, t in g.items()}) for k, (loss, g) in out.items()}))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_equal_one_process():
    mols = molecules()
    want = all_steps(None, mols)
    with socket.socket() as sock:
        sock.bind(("127.0.0.1", 0))
        port = sock.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=100) for _ in procs)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    for name, (loss, grads) in want.items():
        shares = [got[r][name][0] for r in range(2)]
        assert abs(sum(shares) - loss) <= 1e-5 * (abs(loss) + sum(map(abs, shares))) + 1e-7, (name, shares, loss)
        for r in range(2):
            assert got[r][name][1].keys() == grads.keys()
            for n, t in grads.items():
                off = float((torch.from_numpy(got[r][name][1][n]) - t).norm())
                assert off <= 1e-4 * float(t.norm()) + 1e-9, (name, r, n, off, float(t.norm()))
    assert want["nothing"][0] == 0 and not any(t.any() for t in want["nothing"][1].values())
