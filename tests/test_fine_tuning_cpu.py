"""CPU: what two data-parallel ranks (gloo processes) tell each other before a fine-tuning step: counts, atom offsets, and
that one of them refuses its arguments.  The network itself needs a GPU and is not reached."""
import os
import socket
from datetime import timedelta

import pytest
import torch

WORLD = 2


def bare_trainer(group, rank, world):
    """A trainer without a model: the fields that the exchange reads."""
    from diffusion_model_ligandmol_generation_amd.train import ResearchAccurateTrainer
    tr = object.__new__(ResearchAccurateTrainer)
    tr.group = tr.count_group = group
    tr.rank, tr.world, tr.device = rank, world, torch.device("cpu")
    tr.dp_seed_base, tr.step_count = 7, 3
    return tr


class Bag:
    pass


def _refuse_worker(rank, world, port, q, step):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=30))
    tr = bare_trainer(dist.group.WORLD, rank, world)
    out = [tr._over_ranks(lambda: (10 + rank, 5 - rank))]
    # rank 1 brings an odd number of molecules / a rate that is none: whatever the step finds wrong before the network runs
    graph = Bag()
    graph.n_atoms, graph.n_mols = 4, 2

    def inputs(batch, draws):
        if rank == 1:
            raise ValueError("seq_ptr must hold an even number of sequences")
        graph.mol_ptr = torch.tensor([0, 2, 4], dtype=torch.int32)
        return [graph]

    def reached(*a):
        raise AssertionError("the network must not run")

    tr._fine_tune_inputs, tr._atom_type_logits, tr._fine_tune_update = inputs, reached, reached
    from diffusion_model_ligandmol_generation_amd import tokens
    tokens._check_float = lambda t, name: None      # (no GPU here: the one check that asks for one)
    b = Bag()
    b.pos, b.batch, b.atom_types = torch.zeros(4, 3), torch.tensor([0, 0, 1, 1]), torch.zeros(4, dtype=torch.int64)
    call = {"preference": lambda: tr.preference_step(b, None), "policy": lambda: tr.policy_step(b, None, torch.ones(2))}[step]
    try:
        call()
    except Exception as e:
        out.append((type(e).__name__, str(e)))
    out.append(tr._over_ranks(lambda: (1, 1)))      # and both are still in step
    out.append(tr._fine_tune_draws(b, None)["dropout_seed"])
    q.put((rank, out))
    dist.destroy_process_group()


@pytest.mark.parametrize("step", ["preference", "policy"])
def test_a_refusal_reaches_every_rank(step):
    import torch.multiprocessing as mp
    with socket.socket() as sock:
        sock.bind(("127.0.0.1", 0))
        port = sock.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_refuse_worker, args=(r, WORLD, port, q, step)) for r in range(WORLD)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
    assert all(p.exitcode == 0 for p in procs)
    assert got[0][0] == (9, 0) and got[1][0] == (9, 10)         # counts of both, atoms before each
    assert got[0][1] == ("RuntimeError", "1 of 2 ranks refused the arguments of this step")
    assert got[1][1] == ("ValueError", "seq_ptr must hold an even number of sequences")
    assert got[0][2] == (2, 0) and got[1][2] == (2, 1)
    assert got[0][3] == got[1][3] == 10                          # one dropout key for both


def test_one_process():
    tr = bare_trainer(None, 0, 1)
    assert tr._over_ranks(lambda: (10, 4)) == (4, 0)
    with pytest.raises(ValueError, match="mine"):
        tr._over_ranks(lambda: (_ for _ in ()).throw(ValueError("mine")))
