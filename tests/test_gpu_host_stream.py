"""Programs on a context over a host's stream that the host captures into
graphs of its own: what a program keeps between its kernels (packed weights,
attention operands, the folded LayerNorms' statistics) follows what has run,
whatever has been captured and whenever it is replayed."""

import pytest
import torch

import oracle
from beatlm_amd import hip, ir
from tests.blockdata import block_graph, block_values, block_weights

pytestmark = pytest.mark.gpu

T, D, H, MLP, EPS = 257, 384, 6, 1536, 1e-6


class Block:
    """An encoder block over a stream of torch's, and what it should give."""

    def __init__(self, dtype=hip.F32):
        self.stream = torch.cuda.Stream()
        self.ctx = hip.Context(0, stream=self.stream.cuda_stream)
        graph, self.ids = block_graph(T, D, H, MLP, EPS)
        self.prep = ir.prepare(self.ctx, graph)
        self.w = block_weights(D, MLP, 500, "xavier")
        self.x = oracle.normal(1, T * D)
        for tid, v in block_values(self.ids, self.x, self.w).items():
            self.prep.write(tid, v)

    def input(self, seed):
        self.x = oracle.normal(seed, T * D)
        self.prep.write(0, self.x)

    def weight(self, name, seed):
        self.w = dict(self.w, **{name: oracle.xavier(seed, *{"fc1_w": (D, MLP), "qkv_w": (D, 3 * D)}[name])})
        self.prep.write(getattr(self.ids, name), self.w[name])

    def capture(self, first=0, count=None):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=self.stream):
            self.prep.kernels.encode_range(first, len(self.prep.kernels) if count is None else count)
        return graph

    def replay(self, *graphs):
        with torch.cuda.stream(self.stream):
            for g in graphs:
                g.replay()

    def check(self, what):
        got = self.prep.read(self.ids.output)
        bad = oracle.first_mismatch(got, oracle.vit_block(self.x, self.w, T, H, D // H, MLP, EPS))
        assert bad is None, f"{what}: element {bad[0]} is {bad[1]}, the oracle says {bad[2]}"

    def close(self):
        self.prep.close()
        self.ctx.close()


@pytest.fixture
def block(ctx):
    b = Block()
    yield b
    torch.cuda.synchronize()
    b.close()


def test_captured_before_anything_has_run(block):
    """The capture runs nothing: the eager run after it packs the weights itself."""
    graph = block.capture()
    block.prep.run()
    block.check("eager after a capture")
    for seed in (2, 3):
        block.input(seed)
        block.replay(graph)
        block.check("replay")


def test_replays_follow_new_inputs_and_weights(block):
    block.prep.run()
    block.check("eager")
    graph = block.capture()
    for step, (name, seed) in enumerate([(None, 0), ("fc1_w", 900), ("qkv_w", 901), (None, 0)]):
        block.input(10 + step)
        if name:
            block.weight(name, seed)
        block.replay(graph)
        block.check(f"replay {step}")
        block.input(20 + step)
        block.prep.run()
        block.check(f"eager {step}")
        if name:
            block.weight(name, seed + 50)
        block.prep.run()
        block.check(f"eager {step} with another weight")


@pytest.mark.parametrize("cut", [1, 2, 3, 4, 5, 6])
def test_a_program_captured_in_two_parts(block, cut):
    """Each part with the other's work between its replays, and eager work on
    either side."""
    n = len(block.prep.kernels)
    head, tail = block.capture(0, cut), block.capture(cut, n - cut)
    for seed in (30, 31):
        block.input(seed)
        block.replay(head, tail)
        block.check("both parts replayed")
        block.input(seed + 10)
        block.replay(head)
        block.prep.kernels.encode_range(cut, n - cut)
        block.check("the first replayed, the second eager")
        block.input(seed + 20)
        block.prep.kernels.encode_range(0, cut)
        block.replay(tail)
        block.check("the first eager, the second replayed")
        # the program whole for other values, then the tail's replay over a head that ran before it
        block.input(seed + 30)
        for k in range(cut):
            block.prep.kernels.encode(k)
        block.replay(tail)
        block.check("the first kernel by kernel, the second replayed")


def test_a_replay_between_eager_programs(block):
    """The whole program eagerly, and kernel by kernel, after a replay of a part
    that leaves other operands in the scratch."""
    n = len(block.prep.kernels)
    part = block.capture(0, 3)
    for seed in (70, 71):
        block.input(seed)
        block.prep.run()
        block.replay(part)
        block.prep.run()
        block.check("whole")
        block.replay(part)
        for k in range(n):
            block.prep.kernels.encode(k)
        block.check("kernel by kernel")


def test_nothing_is_timed_in_a_capture(block):
    block.prep.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=block.stream):
        block.prep.run()
        with pytest.raises(hip.BackendError) as e:
            block.prep.kernels.time(0, repeats=2)
        assert e.value.code == hip.ERR_INVALID_ARGUMENT
    block.input(80)
    block.replay(graph)
    block.check("the capture around it")
