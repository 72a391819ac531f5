"""A model's answer, token by token: the operators of a serving step together, as a server calls them, on the weights of sky-1
blocks, against the blocks' own forward over the whole sequences."""
import pytest
import torch

from oracle import serve_ref

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
PAGE, VOCAB, LAYERS = 16, 512, 2


class Server:
    """Two decoder blocks, an embedding and a head; a paged cache per layer, page tables and free pages for `requests`."""

    def __init__(self, cdl, requests, longest, heads=4, kv_heads=2, hidden=256):
        self.cdl = cdl
        self.cfg = cdl.sky1.Sky1Config(batch=1, seqlen=longest, hidden=hidden, heads=heads, kv_heads=kv_heads, ffn=512)
        self.params = [{n: p.cuda() for n, p in cdl.sky1.init_params(self.cfg, seed=7 + i, std=0.05).items()} for i in range(LAYERS)]
        gen = torch.Generator(device="cuda").manual_seed(3)
        rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
        self.embedding = rnd(VOCAB, hidden).to(BF16)
        self.head = (rnd(hidden, VOCAB) * 0.2).to(BF16)
        self.table = cdl.sky1.rope_table(longest, 128)
        width = -(-longest // PAGE)
        self.pages = requests * width + 3
        self.caches = [[torch.full((self.pages, PAGE, kv_heads, 128), float("nan"), dtype=BF16, device="cuda") for _ in range(2)]
                       for _ in range(LAYERS)]
        self.block_table = torch.full((requests, width), -1, dtype=I32, device="cuda")
        self.free_pages = torch.randperm(self.pages, generator=gen, device="cuda").to(I32)
        self.free_count = torch.tensor([self.pages], dtype=I32, device="cuda")
        self.cached = torch.zeros(requests, dtype=I32, device="cuda")

    def swiglu(self, gate, up):
        L, act = self.cdl._lib, torch.empty_like(gate)
        L.check(L.packed_lib.cdl_b200_swiglu_fwd(*map(L.tensor_bytes, (gate, up, act)), L.current_stream()))
        return act

    def step(self, tokens, added, prompt):
        """The logits of all rows; tokens i32 [rows], added i32 [requests]."""
        ops, serve, cfg = self.cdl.ops, self.cdl.serve, self.cfg
        rows = tokens.shape[0]
        plan = serve.cache_plan(self.cached, added, self.block_table, self.free_pages, self.free_count,
                                serve.CachePlanOpts(PAGE, self.pages, rows))
        x = self.embedding[tokens.long()]
        h, hk = cfg.heads, cfg.kv_heads
        for p, (k_cache, v_cache) in zip(self.params, self.caches):
            n = ops.norm_fwd(x, ops.NormFwdOpts(scale=p["norm1"])).y
            qkv = ops.matmul(n, p["wqkv"]).view(rows, h + 2 * hk, 128)
            q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
            if prompt:  # q and k rotated where they are: the prompts attend to themselves
                serve.cache_write(k, v, plan.slots, k_cache, v_cache, q=q, table=self.table, positions=plan.positions, q_out=q, k_out=k)
                a = ops.attention_fwd(q, k, v, ops.AttentionOpts(cu_seqlens_q=plan.cu_seqlens, cu_seqlens_k=plan.cu_seqlens)).out
            else:
                w = serve.cache_write(k, v, plan.slots, k_cache, v_cache, q=q, table=self.table, positions=plan.positions)
                a = serve.attention_decode(w.q, k_cache, v_cache, self.block_table, plan.seq_lens).out
            x = ops.matmul(a.reshape(rows, h * 128), p["wo"], ops.MatmulOpts(c=x, beta=1.0))
            n = ops.norm_fwd(x, ops.NormFwdOpts(scale=p["norm2"])).y
            act = self.swiglu(ops.matmul(n, p["wgate"]), ops.matmul(n, p["wup"]))
            x = ops.matmul(act, p["wdown"], ops.MatmulOpts(c=x, beta=1.0))
        self.cached.copy_(plan.seq_lens)
        self.free_count.copy_(plan.free_left)
        return x, ops.matmul(x, self.head, ops.MatmulOpts(out=torch.float32))

    def whole(self, tokens):
        """The last block's output over one sequence, by the blocks' own forward."""
        cfg = self.cdl.sky1.Sky1Config(**{**self.cfg.__dict__, "seqlen": tokens.shape[0]})
        x = self.embedding[tokens.long()].contiguous()
        for p in self.params:
            x = self.cdl.sky1.Sky1Block(cfg, p).forward(x)
        return x


def test_answers_equal_the_whole_forward(cdl, gpu_ok):
    """Prompts of different lengths, then tokens one by one: each step's hidden states against the blocks over all tokens so far.

    Both round to bf16 after every product and norm, at other places of the rotation and of the attention: a few roundings of
    2^-8 of the residual stream per block; 2^-5 of its norm holds them."""
    serve, lens, steps = cdl.serve, [37, 1, 64, 5], 20
    srv = Server(cdl, len(lens), 96)
    gen = torch.Generator(device="cuda").manual_seed(5)
    texts = [torch.randint(0, VOCAB, (n,), generator=gen, device="cuda", dtype=I32) for n in lens]
    added = torch.tensor(lens, dtype=I32, device="cuda")
    x, logits = srv.step(torch.cat(texts), added, prompt=True)
    ends = torch.tensor(lens, device="cuda").cumsum(0) - 1
    hidden = [[r] for r in x.split(lens)]
    logits = logits[ends]
    one = torch.ones_like(added)
    for i in range(steps):
        u = torch.rand(len(lens), generator=gen, device="cuda")
        opts = serve.SampleOpts(temperature=0.8, top_k=[0, 40][i % 2], top_p=[0.9, 1.0][i % 2], min_p=0.01)
        token = serve.sample(logits, u, opts).token
        z = logits.double().cpu().numpy()
        want = [serve_ref.sample(z[b], u[b].item(), 0.8, opts.top_k, opts.top_p, 0.01)[0] for b in range(len(lens))]
        assert token.tolist() == want
        texts = [torch.cat([t, token[b:b + 1]]) for b, t in enumerate(texts)]
        x, logits = srv.step(token, one, prompt=False)
        for b, r in enumerate(x.split(1)):
            hidden[b].append(r)
    assert srv.cached.tolist() == [n + steps for n in lens]
    assert srv.free_count.item() == srv.pages - sum(-(-(n + steps) // PAGE) for n in lens)
    for t, h in zip(texts, hidden):
        ref, got = srv.whole(t).float(), torch.cat(h).float()
        assert got.shape == ref.shape
        assert ((got - ref).norm(dim=1) <= 2.0 ** -5 * ref.norm(dim=1)).all()


def test_a_captured_step_goes_on_by_itself(cdl, gpu_ok):
    """One decoding step captured once: replays read lengths, page tables and free pages on the device, cross page borders and take
    pages, and give the bits of the same steps called one by one."""
    serve, lens, steps = cdl.serve, [14, 31, 3], 40
    results = []
    for captured in (False, True):
        srv = Server(cdl, len(lens), 96)
        gen = torch.Generator(device="cuda").manual_seed(9)
        text = torch.randint(0, VOCAB, (sum(lens),), generator=gen, device="cuda", dtype=I32)
        uniform = torch.rand(steps, len(lens), generator=gen, device="cuda")
        _, logits = srv.step(text, torch.tensor(lens, dtype=I32, device="cuda"), prompt=True)
        logits = logits[torch.tensor(lens, device="cuda").cumsum(0) - 1]
        one = torch.ones(len(lens), dtype=I32, device="cuda")
        state = {"logits": logits.clone(), "u": uniform[0].clone()}

        def step():
            token = serve.sample(state["logits"], state["u"], serve.SampleOpts(top_p=0.95)).token
            _, out = srv.step(token, one, prompt=False)
            state["logits"].copy_(out)
            return token

        tokens = []
        if captured:
            cached, free, table = srv.cached.clone(), srv.free_count.clone(), srv.block_table.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()  # warm-up
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                token = step()
            srv.cached.copy_(cached), srv.free_count.copy_(free), srv.block_table.copy_(table), state["logits"].copy_(logits)
        for i in range(steps):
            state["u"].copy_(uniform[i])
            if captured:
                graph.replay()
                tokens.append(token.clone())
            else:
                tokens.append(step())
        torch.cuda.synchronize()
        results.append((torch.stack(tokens), state["logits"].clone(), srv.cached.clone(), srv.free_count.clone(), srv.block_table.clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][2].tolist() == [n + steps for n in lens]
