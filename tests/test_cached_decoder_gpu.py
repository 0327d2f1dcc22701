"""The operators between the projections as a decoder uses them: QKV projection, cache write, attention, O projection, for a prompt and
for the steps behind it, eagerly and from a graph."""
import pytest
import torch

from breeze_tts_cpp_b200 import ops
from tests.cache_reference import attention, check

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV_HEADS, HEAD_DIM, PAGE, STREAMS, MOST = 256, 4, 2, 64, 16, 3, 6  # MOST: pages of a stream
WIDTHS = (HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM)


class Decoder:
    """One attention block. Its buffers are those of a step of at most `rows` tokens; all of them stay where they are, so that a step can be captured."""

    def __init__(self, mode, rows, stream=None, prefix=0):
        self.stream = stream or torch.cuda.default_stream()
        g = torch.Generator().manual_seed(3)
        new = lambda *shape, std=1.0, mean=0.0: (torch.randn(*shape, generator=g) * std + mean).bfloat16().cuda()  # noqa: E731
        with torch.cuda.stream(self.stream):
            self.ctx = ops.Context(mode, stream=stream, workspace_bytes=32 << 20)
            self.qkv = ops.Linear(self.ctx, [new(n, HIDDEN, std=0.08) for n in WIDTHS], max_rows=rows)
            self.o = ops.Linear(self.ctx, [new(HIDDEN, WIDTHS[0], std=0.08)], max_rows=rows)
            self.q_norm, self.k_norm = new(HEAD_DIM, std=0.1, mean=1.0), new(HEAD_DIM, std=0.1, mean=1.0)
            self.rotary = ops.Rotary.plan(HEAD_DIM, 1e5)
            self.cache = ops.CacheView.empty(STREAMS * MOST + 2 + 4, KV_HEADS, PAGE, HEAD_DIM, ops.format_of(mode))
            order = torch.randperm(STREAMS * MOST + 4, generator=g).to(torch.int32).cuda() + 1
            self.pages, self.prefix_pages = order[: STREAMS * MOST].view(STREAMS, MOST), order[STREAMS * MOST:]
            self.prefix_length = torch.tensor([prefix], dtype=torch.int32, device="cuda") if prefix else None
            for t in (self.cache.key_scales, self.cache.value_scales):
                t.fill_(float("nan"))  # nothing may read what nobody wrote
            self.x = torch.zeros(rows, HIDDEN, dtype=torch.bfloat16, device="cuda")
            self.packed = torch.zeros(rows, sum(WIDTHS), dtype=torch.bfloat16, device="cuda")
            self.out, self.y = torch.zeros(rows, WIDTHS[0], dtype=torch.bfloat16, device="cuda"), torch.zeros_like(self.x)
            self.positions, self.slots = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
            self.lengths, self.offsets = torch.zeros(STREAMS, dtype=torch.int32, device="cuda"), None
            self.stream.synchronize()

    def put(self, x, lengths, counts):
        """The step's tokens, and where they go: the last of each stream's."""
        before = 0 if self.prefix_length is None else int(self.prefix_length)
        tokens = [(b, p) for b in range(STREAMS) for p in range(lengths[b] - counts[b], lengths[b])]
        stream = torch.tensor([b for b, _ in tokens], device="cuda")
        at = torch.tensor([p for _, p in tokens], device="cuda")
        self.x.copy_(x)
        self.positions.copy_(at + before)
        self.slots.copy_(self.pages[stream, at // PAGE] * PAGE + at % PAGE)
        self.lengths.copy_(torch.tensor(lengths))
        self.offsets = None if max(counts) == 1 else torch.tensor([sum(counts[:b]) for b in range(STREAMS + 1)], dtype=torch.int32, device="cuda")

    def step(self):
        self.qkv.forward(self.x, self.packed)
        q, k, v = self.packed.split(WIDTHS, 1)
        self.ctx.cache_write(self.cache, k, v, self.slots, self.positions, self.rotary, q, q, self.q_norm, self.k_norm)
        more = {} if self.prefix_length is None else {"prefix_pages": self.prefix_pages, "prefix_length": self.prefix_length}
        self.ctx.cached_attention(q, self.cache, self.pages, self.lengths, self.out, query_offsets=self.offsets, **more)
        self.o.forward(self.out, self.y)


def moved(to, was):
    """`to` holds what `was` holds: the same cache, pages and weights."""
    for name in ("keys", "values", "key_scales", "value_scales"):
        getattr(to.cache, name).copy_(getattr(was.cache, name))


@pytest.mark.parametrize("prefix", [0, 37])
@pytest.mark.parametrize("mode", ["int8", "fp8", "group_int8"])
def test_prompts_and_steps(mode, prefix):
    g = torch.Generator().manual_seed(5)
    counts, lengths = [30, 7, 18], [30, 7, 18]
    prompt, side = Decoder(mode, sum(counts), prefix=prefix), torch.cuda.Stream()
    captured, eager = Decoder(mode, STREAMS, side, prefix), Decoder(mode, STREAMS, prefix=prefix)
    if prefix:  # the shared tokens, as a prompt of their own left them
        shared = torch.randn(prefix, KV_HEADS * HEAD_DIM, generator=g).bfloat16().cuda()
        at = torch.arange(prefix, device="cuda")
        prompt.ctx.cache_write(prompt.cache, shared, shared.flip(0), (prompt.prefix_pages[at // PAGE] * PAGE + at % PAGE).to(torch.int32))
    prompt.put(torch.randn(sum(counts), HIDDEN, generator=g).bfloat16().cuda(), lengths, counts)
    prompt.step()
    torch.cuda.synchronize()

    def verify(d, counts):
        offsets = [sum(counts[:b]) for b in range(STREAMS + 1)]
        want, bound = attention(d.packed[:, :WIDTHS[0]].cpu(), d.cache, d.pages.cpu(), d.lengths.tolist(), torch.zeros(d.out.shape), None, offsets,
                                d.prefix_pages.cpu() if prefix else None, prefix)
        check(d.out, want, bound)
        assert torch.isfinite(d.y).all() and d.ctx.status() == 0

    verify(prompt, counts)
    moved(captured, prompt)
    moved(eager, prompt)
    torch.cuda.synchronize()
    graph = None
    for step in range(4):
        lengths = [n + 1 for n in lengths]
        x = torch.randn(STREAMS, HIDDEN, generator=g).bfloat16().cuda()
        for d in (captured, eager):
            d.put(x, lengths, [1] * STREAMS)
        torch.cuda.synchronize()
        eager.step()
        if graph is None:
            with torch.cuda.stream(side):
                captured.step()  # loads the kernels; the capture's replay writes the same again
                side.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    captured.step()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        verify(eager, [1] * STREAMS)
        for a, b in ((captured.out, eager.out), (captured.y, eager.y), (captured.cache.keys, eager.cache.keys),
                     (captured.cache.value_scales.nan_to_num(-1.0), eager.cache.value_scales.nan_to_num(-1.0))):
            assert torch.equal(a, b)
    del graph


def test_two_contexts_at_once():
    """A context is one stream's: two of them run at the same time without a shared workspace."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    decoders = [Decoder("int8", STREAMS, s) for s in streams]
    alone = []
    for d in decoders:
        for t in (d.cache.key_scales, d.cache.value_scales):
            t.fill_(0.01)
        d.put(torch.randn(STREAMS, HIDDEN, generator=torch.Generator().manual_seed(7)).bfloat16().cuda(), [80, 65, 90], [1] * STREAMS)
        torch.cuda.synchronize()
        with torch.cuda.stream(d.stream):
            d.step()
        torch.cuda.synchronize()
        alone.append(d.out.clone())
    for _ in range(50):
        for d in decoders:
            with torch.cuda.stream(d.stream):
                d.step()
    torch.cuda.synchronize()
    for d, want in zip(decoders, alone):
        assert torch.equal(d.out, want) and d.ctx.status() == 0
