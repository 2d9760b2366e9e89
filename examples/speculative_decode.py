"""Speculative decoding of a few sequences through full-attention layers: the paged 8-bit cache, its attention, the MoE half and
the verification of drafted tokens in the loop they are made for.

    python examples/speculative_decode.py [--sequences 4] [--layers 2] [--prompt 1000] [--drafts 4] [--steps 16]

Each layer is the model's full-attention layer (16 query heads, 2 key/value heads of 256, 64 of them rotated, a norm of each query's
and key's head before that, an output gate) with random weights; the draft model is a table of next-token probabilities.  The head norm
and the gate are plain torch: the library has neither.  A step feeds every sequence its last token and its
drafts in one call, verifies the drafts against the step's probabilities, and takes the rejected ones back by setting the lengths
to what the verification returns: their keys and values stay in the pages until the next append writes over them.  Nothing in the
loop waits for the GPU."""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from __graft_entry__ import load_package  # noqa: E402

HIDDEN, Q_HEADS, KV_HEADS, HEAD_DIM, ROTARY, PAGE = 2048, 16, 2, 256, 64, 64
THETA = 1.0e7
QUERY_COLUMNS, KV_COLUMNS = Q_HEADS * 2 * HEAD_DIM, KV_HEADS * HEAD_DIM      # a head's query, then its gate


def head_norm(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """Root mean square norm of each head, in FP32."""
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1.0e-6) * (1.0 + weight.float())).bfloat16()


class Model:
    def __init__(self, sequences: int, layers: int, tokens: int, max_rows: int, vocabulary: int = 4096, seed: int = 1) -> None:
        package = load_package()
        self.verify_drafts = package.verify_drafts
        device = torch.device("cuda")
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape: int, std: float = 0.02, dtype=torch.bfloat16):
            return (torch.randn(*shape, generator=g, device=device) * std).to(dtype)

        self.vocabulary, self.layers, self.sequences = vocabulary, layers, sequences
        self.moe = package.MoeProvider(layers=layers, max_prefill_tokens=max_rows)
        for layer in range(layers):
            self.moe.bind_layer(layer, package.synth.layer_weights_cuda_fast(seed, layer, device))
        self.embedding = normal(vocabulary, HIDDEN, std=1.0)
        self.head = normal(vocabulary, HIDDEN, std=0.01)      # flat probabilities, so that a table can draft for it
        self.norms = [torch.zeros(HIDDEN, dtype=torch.bfloat16, device=device) for _ in range(layers + 1)]      # stored less one
        self.qkv = [normal(QUERY_COLUMNS + 2 * KV_COLUMNS, HIDDEN) for _ in range(layers)]
        self.out = [normal(HIDDEN, Q_HEADS * HEAD_DIM) for _ in range(layers)]
        self.head_norms = [(normal(HEAD_DIM, std=0.1), normal(HEAD_DIM, std=0.1)) for _ in range(layers)]      # of q and k, stored less one
        self.draft_table = torch.softmax(normal(vocabulary, vocabulary, std=1.0, dtype=torch.float32), dim=-1)

        columns = (tokens + PAGE - 1) // PAGE
        self.cache = package.KvCache(q_heads=Q_HEADS, kv_heads=KV_HEADS, head_dim=HEAD_DIM, rotary_dim=ROTARY, page_tokens=PAGE,
                                     pages=sequences * columns, layers=layers, max_sequences=sequences)
        self.pages = [self.cache.allocate_layer() for _ in range(layers)]
        for layer, tensors in enumerate(self.pages):
            self.cache.bind_layer(layer, *tensors)
        angle = torch.arange(tokens, dtype=torch.float64)[:, None] * THETA ** (-torch.arange(0, ROTARY, 2, dtype=torch.float64) / ROTARY)
        self.rotation = torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device)
        self.cache.set_rotation(self.rotation)
        # pages in any order
        self.table = torch.randperm(sequences * columns, generator=g, device=device).int().view(sequences, columns)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)

    def projection(self, layer: int, normed: torch.Tensor) -> tuple[torch.Tensor, ...]:
        """q and its gate [tokens, 16, 256], k and v [tokens, 2, 256]; gate and v are views of one product's rows."""
        row = self.moe.gemm(normed, self.qkv[layer])
        q = row[:, :QUERY_COLUMNS].unflatten(1, (Q_HEADS, 2, HEAD_DIM))
        k, v = row[:, QUERY_COLUMNS:].unflatten(1, (2, KV_HEADS, HEAD_DIM)).unbind(1)
        q_norm, k_norm = self.head_norms[layer]
        return head_norm(q[:, :, 0], q_norm), q[:, :, 1], head_norm(k, k_norm), v

    def probabilities(self, tokens: torch.Tensor, all_rows: bool) -> torch.Tensor:
        """Next-token probabilities after the tokens [sequences, new], which go into the cache: FP32 [sequences, rows, vocabulary]."""
        sequences, new = tokens.shape
        self.lengths += new
        batch = self.cache.batch(self.table, self.lengths, tokens=sequences * new)
        x = self.embedding[tokens.reshape(-1).long()]
        _, normed = self.moe.rmsnorm(x, self.norms[0])
        for layer in range(self.layers):
            q, gate, k, v = self.projection(layer, normed)
            q = self.cache.append(layer, batch, k, v, q=q)
            o = self.cache.attention(layer, batch, q) * torch.sigmoid(gate)
            attended = self.moe.gemm(o.view(sequences * new, Q_HEADS * HEAD_DIM), self.out[layer])
            x, normed = self.moe.prefill_fused(attended, x, layer, self.norms[layer + 1])
        normed = normed.view(sequences, new, HIDDEN)
        if not all_rows:
            normed = normed[:, -1:].contiguous()
        logits = self.moe.gemm(normed.view(-1, HIDDEN), self.head).view(sequences, -1, self.vocabulary)
        return torch.softmax(logits.float(), dim=-1)

    def draft(self, last: torch.Tensor, drafts: int, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
        """Tokens [sequences, drafts] drawn one after the other, and the probabilities that each was drawn from."""
        tokens, rows = [], []
        for _ in range(drafts):
            rows.append(self.draft_table[last.long()])
            last = torch.multinomial(rows[-1], 1, generator=g)[:, 0].int()
            tokens.append(last)
        return torch.stack(tokens, 1), torch.stack(rows, 1)

    def release(self) -> None:
        self.cache.release()
        self.moe.release()


def run(model: Model, prompt: torch.Tensor, drafts: int, steps: int, seed: int = 2) -> tuple[torch.Tensor, torch.Tensor]:
    """Returns the drafts accepted [steps, sequences] and the tokens of each step [steps, sequences, drafts + 1], -1 behind the
    one that was drawn."""
    sequences = model.sequences
    g = torch.Generator(device="cuda").manual_seed(seed)
    uniforms = torch.rand(steps + 1, sequences, drafts + 1, generator=g, device="cuda")
    none = torch.empty(sequences, 0, dtype=torch.int32, device="cuda")
    _, first = model.verify_drafts(model.probabilities(prompt, all_rows=False), none, uniforms[steps, :, :1].contiguous())
    last = first[:, 0]
    accepted, tokens = [], []
    for step in range(steps):
        drafted, chances = model.draft(last, drafts, g)
        target = model.probabilities(torch.cat([last[:, None], drafted], 1), all_rows=True)
        a, out, lengths = model.verify_drafts(target, drafted, uniforms[step], draft_probabilities=chances, cache_lengths=model.lengths)
        model.lengths.copy_(lengths)
        last = out.gather(1, a[:, None].long())[:, 0]
        accepted.append(a)
        tokens.append(out)
    model.cache.sync()
    return torch.stack(accepted), torch.cat([torch.full((1, sequences, drafts + 1), -1, dtype=torch.int32, device="cuda").index_copy(
        2, torch.zeros(1, dtype=torch.long, device="cuda"), first[None]), torch.stack(tokens)])


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("sequences", 4), ("layers", 2), ("prompt", 1000), ("drafts", 4), ("steps", 16)):
        parser.add_argument(f"--{name}", type=int, default=default)
    args = parser.parse_args()
    rows = args.sequences * max(args.prompt, args.drafts + 1)
    model = Model(args.sequences, args.layers, args.prompt + (args.steps + 1) * (args.drafts + 1), rows)
    prompt = torch.randint(0, model.vocabulary, (args.sequences, args.prompt), dtype=torch.int32, device="cuda")
    accepted, tokens = run(model, prompt, args.drafts, args.steps)
    for s in range(args.sequences):
        row = [t for t in tokens[:, s].flatten().tolist() if t >= 0]
        print(f"sequence {s}: {len(row)} tokens, {int(accepted[:, s].sum())} of {args.drafts * args.steps} drafts accepted: {row[:12]} ...")
    model.release()


if __name__ == "__main__":
    main()
