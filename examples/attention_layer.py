"""An attention layer over an 8-bit paged cache, prompts in chunks and then token by token, from the framework's own kernels:

    x -> gemm (queries, keys and values in one product) -> rope (queries and keys in one call) -> kvcache_append -> attention_kv8 -> gemm

and several tokens at a time, drafted as a tree of which one path turns out to be right:

    parents -> draft_tree;  x -> gemm -> kvcache_append_rope -> attention_kv8_tree -> gemm;  the path -> kvcache_keep

    python examples/attention_layer.py        # on an MI355X: two prompts, then a captured decode step, or trees; against the same layer in f32
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import __graft_entry__ as ge  # noqa: E402


class AttentionLayer:
    """Weights [out, in] in bf16; a cache of `pages` pages, of which `table` names each sequence's."""

    def __init__(self, pa, width, heads, kv_heads, head_dim, sequences, longest, page_size=64, code_type=None, seed=0):
        self.pa, self.heads, self.kv_heads, self.head_dim, self.sequences = pa, heads, kv_heads, head_dim, sequences
        self.code_type = pa.E4M3 if code_type is None else code_type
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows = (heads + 2 * kv_heads) * head_dim
        self.w_qkv = (torch.randn((rows, width), generator=g, device="cuda") * width ** -0.5).bfloat16()
        self.w_out = (torch.randn((width, heads * head_dim), generator=g, device="cuda") * (heads * head_dim) ** -0.5).bfloat16()
        self.turns = pa.rope_table(longest, head_dim)
        a_sequence = -(-longest // page_size)
        pages = sequences * a_sequence
        self.k, self.v = (torch.zeros((pages, kv_heads, page_size, head_dim), dtype=torch.uint8, device="cuda") for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros((pages, kv_heads), device="cuda") for _ in range(2))
        # (a server's allocator hands pages out as they come: here in a random order)
        self.table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(sequences, a_sequence)

    def __call__(self, x, positions, lengths, cu_tokens=None, max_tokens=None, max_length=0):
        """x [tokens, width]: the new tokens, sequence by sequence; positions [tokens] int32; lengths [sequences] int32, with the new tokens."""
        pa, tokens = self.pa, x.shape[0]
        qkv = pa.gemm(x, self.w_qkv, pa.BF16, pa.BF16).view(tokens, -1, self.head_dim)
        qk = qkv[:, :self.heads + self.kv_heads]
        pa.rope(qk, self.turns, positions, out=qk)
        q, k, v = qk[:, :self.heads], qk[:, self.heads:], qkv[:, self.heads + self.kv_heads:]
        cache = (self.k, self.v, self.k_scale, self.v_scale, self.table, lengths, self.code_type)
        pa.kvcache_append(k, v, *cache, cu_tokens=cu_tokens, max_tokens=max_tokens)
        o = pa.attention_kv8(q, *cache, cu_tokens=cu_tokens, max_tokens=max_tokens, max_length=max_length)
        return pa.gemm(o.view(tokens, -1), self.w_out, pa.BF16, pa.BF16)

    def drafted(self, x, tree, lengths, cu_tokens=None, max_tokens=None, max_length=0):
        """x [tokens, width]: drafted tokens, sequence by sequence; tree: their rows of draft_tree(); lengths [sequences] int32, with them."""
        pa, tokens = self.pa, x.shape[0]
        qkv = pa.gemm(x, self.w_qkv, pa.BF16, pa.BF16).view(tokens, -1, self.head_dim)
        q, k, v = qkv[:, :self.heads], qkv[:, self.heads:self.heads + self.kv_heads], qkv[:, self.heads + self.kv_heads:]
        cache = (self.k, self.v, self.k_scale, self.v_scale, self.table, lengths, self.code_type)
        pa.kvcache_append_rope(q, k, v, *cache, self.turns, tree=tree, cu_tokens=cu_tokens, max_tokens=max_tokens, out=q)
        o = pa.attention_kv8_tree(q, *cache, tree, cu_tokens=cu_tokens, max_tokens=max_tokens, max_length=max_length)
        return pa.gemm(o.view(tokens, -1), self.w_out, pa.BF16, pa.BF16)

    def keep(self, kept, lengths, max_tokens, cu_tokens=None):
        """The lengths with the path `kept` [sequences, most] of the drafted tokens alone, which the cache then holds behind what is older."""
        return self.pa.kvcache_keep(kept, self.k, self.v, self.k_scale, self.v_scale, self.table, lengths, self.code_type, cu_tokens=cu_tokens,
                                    max_tokens=max_tokens)

    def plain(self, x):
        """One sequence's x [tokens, width] from its first token on, in f32, without a cache."""
        tokens, d = x.shape[0], self.head_dim
        qkv = (x.float() @ self.w_qkv.float().T).view(tokens, -1, d)
        qk, v = qkv[:, :self.heads + self.kv_heads], qkv[:, self.heads + self.kv_heads:]
        cos, sin = self.turns[:tokens, None, :d // 2], self.turns[:tokens, None, d // 2:]
        lo, hi = qk[..., :d // 2], qk[..., d // 2:]
        qk = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)
        share = self.heads // self.kv_heads
        k, v = (t.repeat_interleave(share, dim=1) for t in (qk[:, self.heads:], v))
        scores = torch.einsum("qhd,khd->hqk", qk[:, :self.heads], k) / math.sqrt(d)
        scores.masked_fill_(torch.ones((tokens, tokens), device="cuda", dtype=torch.bool).triu(1), -math.inf)
        return torch.einsum("hqk,khd->qhd", scores.softmax(dim=-1), v).reshape(tokens, -1) @ self.w_out.float().T


def serve(layer, prompts, chunk, steps):
    """The prompts in chunks of up to `chunk` tokens, ragged; then `steps` tokens each of a captured step.  x of every token comes from `prompts`
    [tokens, width] of each sequence, of which the last `steps` are the decoded ones.  Returns each sequence's outputs."""
    counts = [p.shape[0] - steps for p in prompts]
    outs, done = [[] for _ in prompts], [0] * len(prompts)
    while any(d < n for d, n in zip(done, counts)):
        new = [min(chunk, n - d) for d, n in zip(done, counts)]
        starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        x = torch.cat([p[d:d + n] for p, d, n in zip(prompts, done, new)])
        positions = torch.cat([torch.arange(d, d + n, dtype=torch.int32) for d, n in zip(done, new)]).cuda()
        done = [d + n for d, n in zip(done, new)]
        y = layer(x, positions, torch.tensor(done, dtype=torch.int32, device="cuda"), starts.cuda(), max(new), max(done))
        for s, o in enumerate(outs):
            o.append(y[starts[s]:starts[s + 1]])

    x = torch.zeros((len(prompts), prompts[0].shape[1]), dtype=torch.bfloat16, device="cuda")
    lengths = torch.tensor(done, dtype=torch.int32, device="cuda")
    positions, one = lengths.clone(), torch.ones_like(lengths)
    graph = None
    for step in range(steps):
        x.copy_(torch.stack([p[n + step] for p, n in zip(prompts, counts)]))
        lengths += one
        if graph is None:  # (kernels only: a replay reads the lengths and positions that are there then)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = layer(x, positions, lengths)
        graph.replay()
        positions += one
        for s, o in enumerate(outs):
            o.append(y[s:s + 1].clone())
    return [torch.cat(o) for o in outs]


def serve_drafted(layer, prompts, known, chunk, drafted, seed=0):
    """The first `known` tokens of each prompt in chunks, then trees of `drafted` tokens each, one path of which holds the sequence's next tokens: what a
    server's drafter gives, and its model then finds right.  Returns each sequence's outputs of the tokens that were kept."""
    rng = random.Random(seed)
    outs = serve(layer, [p[:known] for p in prompts], chunk, 0)
    done, pa = [known] * len(prompts), layer.pa
    lengths = torch.tensor(done, dtype=torch.int32, device="cuda")
    while any(d < p.shape[0] for d, p in zip(done, prompts)):
        new = [drafted if d < p.shape[0] else 0 for d, p in zip(done, prompts)]
        starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        parents, paths, x = [], [], []
        for s, p in enumerate(prompts):
            mine = [rng.randrange(-1, i) for i in range(new[s])]
            path, at = [], rng.randrange(new[s]) if mine else -1
            while at >= 0:
                path.insert(0, at)
                at = mine[at]
            path = path[:p.shape[0] - done[s]]
            wrong = torch.randn((new[s], p.shape[1]), generator=torch.Generator().manual_seed(rng.randrange(1 << 30))).to(p)
            wrong[path] = p[done[s]:done[s] + len(path)]
            parents += mine
            paths.append(path)
            x.append(wrong)
        cu = starts.cuda()
        tree = pa.draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), len(prompts), cu_tokens=cu, max_tokens=drafted)
        lengths += cu[1:] - cu[:-1]
        y = layer.drafted(torch.cat(x), tree, lengths, cu, drafted, max(done) + drafted)
        most = max(len(path) for path in paths)
        kept = torch.tensor([path + [-1] * (most - len(path)) for path in paths], dtype=torch.int32, device="cuda").view(len(prompts), most)
        lengths = layer.keep(kept, lengths, drafted, cu)
        for s, path in enumerate(paths):
            outs[s] = torch.cat([outs[s], y[int(starts[s]):int(starts[s + 1])][path]])
            done[s] += len(path)
    return outs


def relative_error(layer, prompts, outs):
    """The largest over sequences of |out - plain| / |plain|, both over all tokens."""
    return max(float((o.float() - layer.plain(p)).norm() / layer.plain(p).norm()) for o, p in zip(outs, prompts))


def main():
    pa = ge.load_package()
    pa.init(0)
    for code, name in ((pa.E4M3, "e4m3"), (pa.I8, "int8")):
        layer = AttentionLayer(pa, width=1024, heads=16, kv_heads=4, head_dim=128, sequences=2, longest=1024, code_type=code)
        g = torch.Generator(device="cuda").manual_seed(1)
        prompts = [torch.randn((n, 1024), generator=g, device="cuda").bfloat16() for n in (700, 333)]
        outs = serve(layer, prompts, chunk=256, steps=8)
        print(f"{name} cache: relative error {relative_error(layer, prompts, outs):.4f} over {sum(p.shape[0] for p in prompts)} tokens")
        outs = serve_drafted(layer, prompts, known=300, chunk=256, drafted=24)
        print(f"{name} cache, drafted trees: relative error {relative_error(layer, prompts, outs):.4f}")


if __name__ == "__main__":
    main()
