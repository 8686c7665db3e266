"""Calls of attention and the cache in HIP graphs that outlive what they were captured with: plans that are dropped, a
workspace that larger calls outgrow; and what cannot be captured."""
import pytest
import torch

from test_kv_cache_gpu import Filled, bits, rand

pytestmark = pytest.mark.gpu


class Case:
    """Calls whose plans are all in device memory: 200 sequences' tokens, prompts, rows in several parts."""

    def __init__(self, cvs, stream):
        self.ctx = cvs.Context(0, stream=stream.cuda_stream)
        self.f = Filled(self.ctx, 1, 900, 32, 2, 64, "bf16")
        (root,) = self.f.new()
        self.f.append([root], [9000])
        self.seqs = self.f.fork(root, 200)
        self.f.append(self.seqs, [1 + i % 5 for i in range(200)])
        self.q, self.k, self.v = (rand(i, 200, h, 64, dtype="bf16") for i, h in enumerate((8, 2, 2)))
        self.outs = [torch.empty_like(x) for x in (self.q, self.q, self.k, self.v)]

    def plans(self, shift=0):
        """Other plans of the same sizes for another shift."""
        seqs = self.seqs[shift:] + self.seqs[:shift]
        return self.f.cache.plan(seqs, [1] * 200, heads=8), self.ctx.prompt_plan([3 + shift, 100 - shift, 97], 8, 2)

    def calls(self, step, prompt):
        self.f.cache.attention_async(step, self.q, self.outs[0])
        self.ctx.prompt_attention_async(prompt, self.q, self.k, self.v, self.outs[1])
        self.f.cache.read_async(step, self.outs[2], self.outs[3])

    def capture(self, stream, plans):
        self.calls(*plans)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            self.calls(*plans)
        return graph

    def check(self, stream, graph, want):
        for seed in range(3):
            for x in self.outs:
                x.fill_(9.0)
            graph.replay()
            stream.synchronize()
            for x, y in zip(self.outs, want):
                assert torch.equal(bits(x), bits(y)), seed
            torch.randn(1000, 1000, device="cuda").sum().item()


def test_plans_dropped_before_a_replay(cvs):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = Case(cvs, stream)
        plans = c.plans()
        graph = c.capture(stream, plans)
        c.calls(*plans)
        want = [x.clone() for x in c.outs]
        del plans
        others = [c.plans(shift) for shift in (1, 7, 50)]  # not in the captured plans' memory
        for p in others:
            c.calls(*p)
        c.check(stream, graph, want)
        del others
        c.calls(*c.plans())
        for x, y in zip(c.outs, want):
            assert torch.equal(bits(x), bits(y))
        c.f.cache.close()
        c.ctx.close()


def test_a_workspace_outgrown_before_a_replay(cvs):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = Case(cvs, stream)
        plans = c.plans()
        graph = c.capture(stream, plans)
        c.calls(*plans)
        want = [x.clone() for x in c.outs]
        q = rand(9, 200, 64, 64, dtype="bf16")
        big, out = c.f.cache.plan(c.seqs, [1] * 200, heads=64), torch.empty_like(q)
        c.f.cache.attention_async(big, q, out)  # 8 times the parts
        filler = torch.full((1 << 26,), float("nan"), device="cuda")  # where freed memory would be
        c.check(stream, graph, want)
        c.f.cache.attention_async(big, q, out.zero_())
        assert torch.isfinite(out.float()).all()
        del filler
        c.f.cache.close()
        c.ctx.close()


def test_what_cannot_be_captured(cvs):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = Case(cvs, stream)
        cache, plans = c.f.cache, c.plans()
        (kid,) = c.f.fork(c.seqs[0], 1)
        before = cache.pages([kid, *c.seqs]).tolist()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        refused = []
        with torch.cuda.graph(graph, stream=stream):
            for call in (lambda: cache.plan(c.seqs, [1] * 200, heads=8), lambda: c.ctx.prompt_plan([5], 8, 2),
                         lambda: cache.extend([kid], [1]), lambda: cache.compact(),
                         lambda: cache.attention_async(plans[0], c.q, c.outs[0])):
                try:
                    call()
                except ValueError as e:
                    refused.append(str(e))
            c.ctx.prompt_attention_async(plans[1], c.q, c.k, c.v, c.outs[1])
        assert len(refused) == 5 and all("captured" in m for m in refused), refused
        assert "make the call once before" in refused[-1]
        assert cache.pages([kid, *c.seqs]).tolist() == before
        c.outs[1].zero_()
        graph.replay()
        got = c.outs[1].clone()
        c.ctx.prompt_attention_async(plans[1], c.q, c.k, c.v, c.outs[1])
        assert torch.equal(bits(got), bits(c.outs[1]))
        cache.extend([kid], [1])
        cache.compact()
        cache.close()
        c.ctx.close()


def test_captured_on_torchs_stream_with_a_context_of_its_own(cvs):
    """The context's stream joins the capture by the events that order it with torch's."""
    q, k, v = (rand(i, 90, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    out, want = torch.empty_like(q), torch.empty_like(q)
    with cvs.Context(0) as ctx:
        plan = ctx.prompt_plan([40, 50], 4, 2)
        ctx.prompt_attention_async(plan, q, k, v, want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ctx.prompt_attention_async(plan, q * 1, k * 1, v * 1, out)
            doubled = out * 2
        for seed in (0, 20, 40):
            for i, x in enumerate((q, k, v)):
                x.copy_(rand(seed + i, *x.shape, dtype="fp16"))
            ctx.prompt_attention_async(plan, q, k, v, want)
            out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(bits(out), bits(want)) and torch.equal(bits(doubled), bits(want * 2)), seed
