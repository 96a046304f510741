"""A module's dropout bits (hyperconnections_b200.drop_state) under recomputation:
on the CPU the draws themselves, by a stand-in for dropout that computes with
the (seed, offset) it is given; on the GPU the layers and the embedding's
dropout, whose gradients under a checkpoint are those of the plain step."""

import copy
import os
import socket
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
import torch.nn as nn
from torch.utils.checkpoint import checkpoint

from hyperconnections_b200.drop_state import DropState


class Stand(nn.Module):
    """x times what its draw says, so that the gradient shows the draw of the forward that made it."""

    def __init__(self):
        super().__init__()
        self.bits = DropState()
        self.bits.state.copy_(torch.tensor([3, 100]))
        self.seen = []

    def forward(self, x):
        with self.bits.drawn(x.device) as seed:
            self.seen.append(seed.tolist())
            return x * seed[1].to(x.dtype)


def grad_of(out, x):
    return torch.autograd.grad(out.sum(), x)[0].item()


def test_a_plain_step_draws_the_next_offset_and_leaves_the_generator_alone():
    m, x = Stand(), torch.ones(1, requires_grad=True)
    before = torch.get_rng_state()
    assert [grad_of(m(x), x) for _ in range(3)] == [100, 101, 102]
    assert torch.equal(before, torch.get_rng_state()) and m.bits.state.tolist() == [3, 103]


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint(reentrant):
    """Two modules in a segment, one of them twice; two micro-batches, whose backward passes come in either order."""
    for order in ((0, 1), (1, 0)):
        a, b = Stand(), Stand()
        b.bits.state.copy_(torch.tensor([3, 7]))
        x = torch.ones(1, requires_grad=True)
        outs = [checkpoint(lambda t: a(b(a(t))), x, use_reentrant=reentrant) for _ in range(2)]
        want = [100 * 7 * 101, 102 * 8 * 103]
        assert [o.item() for o in outs] == want
        assert a.bits.state.tolist() == [3, 104] and b.bits.state.tolist() == [3, 9]
        for i in order:
            x.grad = None
            outs[i].sum().backward()
            assert x.grad.item() == want[i]
        assert a.bits.state.tolist() == [3, 104] and b.bits.state.tolist() == [3, 9]


def test_checkpoint_inside_a_checkpoint_and_a_graph_kept():
    a, b = Stand(), Stand()
    b.bits.state.copy_(torch.tensor([3, 7]))
    x = torch.ones(1, requires_grad=True)

    def outer(t):
        return a(checkpoint(lambda u: b(u) * b(u), t, use_reentrant=False))

    out = checkpoint(outer, x, use_reentrant=False)
    assert out.item() == 100 * 7 * 8
    for _ in range(2):
        assert torch.autograd.grad(out.sum(), x, retain_graph=True)[0].item() == 2 * 100 * 7 * 8
    assert a.bits.state.tolist() == [3, 101] and b.bits.state.tolist() == [3, 9]


def test_a_step_that_starts_from_the_same_seed_again():
    """The generator reset before every step: each step's backward pass has that step's bits."""
    a, x = Stand(), torch.ones(1, requires_grad=True)
    for k in range(3):
        torch.manual_seed(0)
        assert grad_of(checkpoint(a, x, use_reentrant=False), x) == 100 + k


@pytest.mark.parametrize("reentrant", [False, True])
def test_refusals(reentrant):
    a, x = Stand(), torch.ones(1, requires_grad=True)
    out = checkpoint(a, x, use_reentrant=reentrant, preserve_rng_state=False)
    with pytest.raises(RuntimeError, match="first forward is not known"):
        out.sum().backward()
    outs = []
    for _ in range(2):
        torch.manual_seed(5)
        outs.append(checkpoint(a, x, use_reentrant=reentrant))
    with pytest.raises(RuntimeError, match="two first forwards"):
        outs[0].sum().backward()
    # more draws of the module than it files
    a.bits.KEPT = 4
    outs = [checkpoint(a, x, use_reentrant=reentrant) for _ in range(5)]
    with pytest.raises(RuntimeError, match="first forward is not known"):
        outs[0].sum().backward()
    outs[1].sum().backward()


def test_copies_have_their_own_draws():
    a, x = Stand(), torch.ones(1, requires_grad=True)
    out = checkpoint(a, x, use_reentrant=False)
    b = copy.deepcopy(a)
    assert len(a.bits._filed) == 1 and not b.bits._filed and b.bits.state.tolist() == [3, 101]
    assert not b.state_dict()
    assert grad_of(out, x) == 100


def test_the_state_goes_with_its_module():
    a = Stand()
    a.bits.state.copy_(torch.tensor([1 << 61, 1 << 60]))
    for moved in (a.double(), a.half(), a.to("cpu", torch.bfloat16), a.to_empty(device="cpu"), a.to("meta"), a.cpu()):
        assert moved.bits.state.dtype == torch.int64 and moved.bits.state.tolist() == [1 << 61, 1 << 60]
    with torch.device("meta"):
        made = DropState()
    assert made.state.device.type == "cpu" and made.state[0] != 0
    assert not dict(a.named_buffers()) and not dict(a.named_parameters())
    assert DropState(seeded=False).state.tolist() == [0, 0]


def test_every_rank_has_a_seed_of_its_own(monkeypatch):
    import hyperconnections_b200.drop_state as ds

    for first in (0, 1, 2):  # seeds of the generator
        seeds = []
        for rank in [*range(64), 1000, 4095, 1 << 20]:
            monkeypatch.setattr(ds, "_rank", lambda: rank)
            torch.manual_seed(first)
            seeds.append(DropState().state.tolist())
        assert len({s for s, _ in seeds}) == len(seeds)
        assert all(0 <= s < 1 << 62 and o == 0 for s, o in seeds)


def test_the_state_of_a_layer_can_be_set():
    from tests.test_block_layers import CGHC, FULL, layer

    lay = layer(CGHC, 4, 2, 16, FULL)
    lay.block.drop_state = torch.tensor([5, 6])
    assert lay.block.bits.state.tolist() == [5, 6]
    lay.block.drop_state.copy_(torch.tensor([7, 8]))
    assert lay.block.drop_state.tolist() == [7, 8] and not any("state" in k for k in lay.state_dict())


def test_a_draw_without_autograd_leaves_a_state_that_moves_on():
    m, x = Stand(), torch.ones(1, requires_grad=True)
    with torch.inference_mode():
        m.float()
        m(torch.ones(1))
    with torch.no_grad():
        m(x)
    assert grad_of(m(x), x) == 102


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=60))
    try:
        torch.manual_seed(0)

        class Net(nn.Module):
            def __init__(self):
                super().__init__()
                self.drop, self.fc = Stand(), nn.Linear(4, 4)
                self.drop.bits = DropState()

            def forward(self, x):
                return self.fc(self.drop(x))

        net = nn.parallel.DistributedDataParallel(Net())
        states = [net.module.drop.bits.state.tolist()]
        for _ in range(2):
            net(torch.ones(2, 4)).sum().backward()
            states.append(net.module.drop.bits.state.tolist())
        q.put((rank, states, net.module.drop.seen, net.module.fc.weight.detach().sum().item()))
    finally:
        dist.destroy_process_group()


def test_ranks_that_seed_alike_draw_other_bits():
    """Two ranks build the same model from the same seed: their states differ from the beginning and after forwards of
    DistributedDataParallel; rank 0 has what one process alone has."""
    world = 2
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = sorted(q.get(timeout=120) for _ in range(world))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    torch.manual_seed(0)
    Stand(), nn.Linear(4, 4)
    alone = DropState().state[0].item()
    (_, first, seen0, w0), (_, second, seen1, w1) = res
    assert w0 == w1
    assert first == [[alone, k] for k in range(3)] and seen0 == [[alone, 0], [alone, 1]]
    other = second[0][0]
    assert other != alone and 0 <= other < 1 << 62
    assert second == [[other, k] for k in range(3)] and seen1 == [[other, 0], [other, 1]]


# --------------------------------------------------------------------- GPU
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("name", ["cghc", "ghc", "mhc"])
def test_layer_under_a_checkpoint(name, reentrant):
    """Two layers with every block option in one segment: loss and gradients of the plain step, bit for bit."""
    cuda()
    from tests.test_block_layers import CGHC, FULL, GHC, MHC, layer

    cls = {"cghc": CGHC, "ghc": GHC, "mhc": MHC}[name]
    net = nn.Sequential(layer(cls, 4, 2, 96, FULL), layer(cls, 4, 2, 96, FULL)).cuda()
    x, g = (torch.randn(3, 40, 192, device="cuda") for _ in range(2))

    def step(run):
        for i, lay in enumerate(net):
            lay.block.drop_state.copy_(torch.tensor([77 + i, 5]))
        net.zero_grad(set_to_none=True)
        leaf = x.clone().requires_grad_(True)
        outs = [run(leaf) for _ in range(2)]  # two micro-batches before their backward passes
        for out in outs:
            out.backward(g)
        assert [lay.block.drop_state.tolist() for lay in net] == [[77, 7], [78, 7]]
        return [*(o.detach() for o in outs), leaf.grad, *(p.grad for p in net.parameters() if p.grad is not None)]

    plain = step(net)
    again = step(lambda t: checkpoint(net, t, use_reentrant=reentrant))
    assert not torch.equal(plain[0], plain[1])  # other bits
    assert len(plain) == len(again) and all(torch.equal(a, b) for a, b in zip(plain, again))


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_embedding_dropout_under_a_checkpoint(reentrant):
    cuda()
    from e2e_models import EmbeddingDropout

    drop = EmbeddingDropout(0.5).cuda()
    x = torch.randn(7, 333, device="cuda", requires_grad=True)
    y = checkpoint(drop, x, use_reentrant=reentrant)
    y.backward(torch.ones_like(y))
    assert torch.equal(x.grad != 0, y.detach() != 0)


@pytest.mark.gpu
def test_checkpointed_step_in_a_graph():
    """A step whose forward is run again, captured once: every replay has other bits, and its gradient those of its
    forward."""
    cuda()
    from hyperconnections_b200.ops import hc_dropout

    bits = DropState().cuda()
    x = torch.randn(4000, device="cuda", requires_grad=True)

    def dropped(t):
        with bits.drawn(t.device) as seed:
            return hc_dropout(t, 0.5, seed)

    def step():  # as a checkpoint does: without gradients first, then again inside the backward pass
        class Twice(torch.autograd.Function):
            @staticmethod
            def forward(ctx, t):
                ctx.save_for_backward(t)
                ctx.rng = torch.get_rng_state()
                return dropped(t)

            @staticmethod
            def backward(ctx, g):
                (t,) = ctx.saved_tensors
                after = torch.get_rng_state()
                torch.set_rng_state(ctx.rng)
                with torch.enable_grad():
                    leaf = t.detach().requires_grad_(True)
                    out = dropped(leaf)
                torch.set_rng_state(after)
                return torch.autograd.grad(out, leaf, g)[0]

        y = Twice.apply(x)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(x))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = step()
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gx != 0, y != 0)
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
