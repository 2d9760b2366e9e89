"""Speculative decoding of a few sequences through the model's two kinds of layers: the paged 8-bit cache with its attention, the
convolution and the gated delta rule of the linear-attention layers, the MoE half and the verification of drafted tokens in the loop
they are made for.

    python examples/speculative_decode.py [--sequences 4] [--layers 2] [--linear 3] [--prompt 1000] [--drafts 4] [--steps 16]

A full-attention layer (16 query heads, 2 key/value heads of 256, 64 of them rotated, a norm of each query's and key's head before
that, an output gate) comes after every `linear` linear-attention layers (16 key heads and 32 value heads of 128, a convolution over
four positions, a gated norm), all with random weights; the draft model is a table of next-token probabilities.  A step feeds every
sequence its last token and its drafts in one call, verifies the drafts against the step's probabilities, and takes the rejected ones
back.  The cache does that by its lengths, which are set to what the verification returns: the keys and values of rejected drafts stay
in the pages until the next append writes over them.  The states of the linear-attention layers cannot go back, so none of the step's
tokens enters them at first; those that stand do in a second call, once their number is known.  Nothing in the loop waits for the GPU."""
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
K_HEADS, V_HEADS, LINEAR_DIM, CONV_WIDTH = 16, 32, 128, 4
CHANNELS = (2 * K_HEADS + V_HEADS) * LINEAR_DIM                              # queries, keys and values; then the gates, b and a


class Model:
    def __init__(self, sequences: int, layers: int, tokens: int, max_rows: int, vocabulary: int = 4096, seed: int = 1, linear: int = 0) -> None:
        package = load_package()
        self.verify_drafts, self.head_norm = package.verify_drafts, package.head_norm
        device = torch.device("cuda")
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape: int, std: float = 0.02, dtype=torch.bfloat16):
            return (torch.randn(*shape, generator=g, device=device) * std).to(dtype)

        self.vocabulary, self.sequences = vocabulary, sequences
        # (whether it is a linear-attention layer, which one of its kind)
        self.layers = [(kind < linear, group * linear + kind if kind < linear else group) for group in range(layers) for kind in range(linear + 1)]
        self.moe = package.MoeProvider(layers=len(self.layers), max_prefill_tokens=max_rows)
        for layer in range(len(self.layers)):
            self.moe.bind_layer(layer, package.synth.layer_weights_cuda_fast(seed, layer, device))
        self.embedding = normal(vocabulary, HIDDEN, std=1.0)
        self.head = normal(vocabulary, HIDDEN, std=0.01)      # flat probabilities, so that a table can draft for it
        self.norms = [torch.zeros(HIDDEN, dtype=torch.bfloat16, device=device) for _ in range(len(self.layers) + 1)]      # stored less one
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
        self.linear_count = layers * linear
        if linear:
            self.linear = package.LinearAttention(k_heads=K_HEADS, v_heads=V_HEADS, conv_width=CONV_WIDTH, slots=sequences, layers=self.linear_count,
                                                  max_sequences=sequences, max_tokens=max_rows)
            self.linear_in = [normal(CHANNELS + V_HEADS * LINEAR_DIM + 2 * V_HEADS, HIDDEN) for _ in range(self.linear_count)]
            self.linear_out = [normal(HIDDEN, V_HEADS * LINEAR_DIM) for _ in range(self.linear_count)]
            self.states = [self.linear.allocate_layer() for _ in range(self.linear_count)]
            self.linear_weights = []
            for layer, (conv_states, states) in enumerate(self.states):
                step = torch.empty(V_HEADS, device=device).uniform_(0.001, 0.1, generator=g)
                weights = dict(conv_weight=normal(CHANNELS, CONV_WIDTH, std=0.5), a_log=torch.empty(V_HEADS, device=device).uniform_(0.01, 16.0, generator=g).log(),
                               dt_bias=torch.log(torch.expm1(step)), norm_weight=normal(LINEAR_DIM, std=0.1) + 1.0)
                self.linear.bind_layer(layer, conv_states=conv_states, states=states, **weights)
                self.linear_weights.append(weights)
        self.slots = torch.arange(sequences, dtype=torch.int32, device=device)
        self.nothing = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.pending = []                    # what the linear-attention layers made of a step's tokens
        # pages in any order
        self.table = torch.randperm(sequences * columns, generator=g, device=device).int().view(sequences, columns)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)

    def projection(self, layer: int, normed: torch.Tensor) -> tuple[torch.Tensor, ...]:
        """q and its gate [tokens, 16, 256], k and v [tokens, 2, 256]; gate and v are views of one product's rows."""
        row = self.moe.gemm(normed, self.qkv[layer])
        q = row[:, :QUERY_COLUMNS].unflatten(1, (Q_HEADS, 2, HEAD_DIM))
        k, v = row[:, QUERY_COLUMNS:].unflatten(1, (2, KV_HEADS, HEAD_DIM)).unbind(1)
        q_norm, k_norm = self.head_norms[layer]
        return self.head_norm(q[:, :, 0], q_norm, offset=1.0), q[:, :, 1], self.head_norm(k, k_norm, offset=1.0), v

    def full_attention(self, layer: int, batch, normed: torch.Tensor) -> torch.Tensor:
        q, gate, k, v = self.projection(layer, normed)
        q = self.cache.append(layer, batch, k, v, q=q)
        o = self.head_norm(self.cache.attention(layer, batch, q), gate=gate, activation="sigmoid")
        return self.moe.gemm(o.view(-1, Q_HEADS * HEAD_DIM), self.out[layer])

    def linear_attention(self, layer: int, batch, normed: torch.Tensor) -> torch.Tensor:
        row = self.moe.gemm(normed, self.linear_in[layer])
        x, z, b, a = row.split([CHANNELS, V_HEADS * LINEAR_DIM, V_HEADS, V_HEADS], dim=1)
        q, k, v = self.linear.conv(layer, batch, x).unflatten(1, (-1, LINEAR_DIM)).split([K_HEADS, K_HEADS, V_HEADS], dim=1)
        if batch.keep is not None:
            self.pending.append((x, q, k, v, a, b))
        o = self.linear.delta(layer, batch, q, k, v, a, b, gate=z.unflatten(1, (V_HEADS, LINEAR_DIM)))
        return self.moe.gemm(o.view(-1, V_HEADS * LINEAR_DIM), self.linear_out[layer])

    def linear_batch(self, tokens: int, keep: torch.Tensor | None):
        return self.linear.batch(self.slots, tokens=tokens, lengths=self.lengths, keep=keep) if self.linear_count else None

    def probabilities(self, tokens: torch.Tensor, all_rows: bool, drafted: bool = False) -> torch.Tensor:
        """Next-token probabilities after the tokens [sequences, new], which go into the cache, and into the states unless they are
        drafted: FP32 [sequences, rows, vocabulary]."""
        sequences, new = tokens.shape
        self.lengths += new
        self.pending.clear()
        batch = self.cache.batch(self.table, self.lengths, tokens=sequences * new)
        linear_batch = self.linear_batch(sequences * new, self.nothing if drafted else None)
        x = self.embedding[tokens.reshape(-1).long()]
        _, normed = self.moe.rmsnorm(x, self.norms[0])
        for layer, (linear, which) in enumerate(self.layers):
            attended = self.linear_attention(which, linear_batch, normed) if linear else self.full_attention(which, batch, normed)
            x, normed = self.moe.prefill_fused(attended, x, layer, self.norms[layer + 1])
        normed = normed.view(sequences, new, HIDDEN)
        if not all_rows:
            normed = normed[:, -1:].contiguous()
        logits = self.moe.gemm(normed.view(-1, HIDDEN), self.head).view(sequences, -1, self.vocabulary)
        return torch.softmax(logits.float(), dim=-1)

    def keep(self, kept: torch.Tensor) -> None:
        """Brings the first `kept` (int32 [sequences]) of the last step's tokens into the states, before the lengths change."""
        if self.linear_count:
            batch = self.linear_batch(self.pending[0][0].shape[0], kept)
            for layer, (x, q, k, v, a, b) in enumerate(self.pending):
                self.linear.conv(layer, batch, x)
                self.linear.delta(layer, batch, q, k, v, a, b, outputs=False)

    def draft(self, last: torch.Tensor, drafts: int, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
        """Tokens [sequences, drafts] drawn one after the other, and the probabilities that each was drawn from."""
        tokens, rows = [], []
        for _ in range(drafts):
            rows.append(self.draft_table[last.long()])
            last = torch.multinomial(rows[-1], 1, generator=g)[:, 0].int()
            tokens.append(last)
        return torch.stack(tokens, 1), torch.stack(rows, 1)

    def sync(self) -> None:
        """Waits, and raises if a batch was out of range."""
        self.cache.sync()
        if self.linear_count:
            self.linear.sync()

    def release(self) -> None:
        self.cache.release()
        if self.linear_count:
            self.linear.release()
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
        target = model.probabilities(torch.cat([last[:, None], drafted], 1), all_rows=True, drafted=True)
        a, out, lengths = model.verify_drafts(target, drafted, uniforms[step], draft_probabilities=chances, cache_lengths=model.lengths)
        model.keep(a + 1)
        model.lengths.copy_(lengths)
        last = out.gather(1, a[:, None].long())[:, 0]
        accepted.append(a)
        tokens.append(out)
    model.sync()
    return torch.stack(accepted), torch.cat([torch.full((1, sequences, drafts + 1), -1, dtype=torch.int32, device="cuda").index_copy(
        2, torch.zeros(1, dtype=torch.long, device="cuda"), first[None]), torch.stack(tokens)])


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("sequences", 4), ("layers", 2), ("linear", 3), ("prompt", 1000), ("drafts", 4), ("steps", 16)):
        parser.add_argument(f"--{name}", type=int, default=default)
    args = parser.parse_args()
    rows = args.sequences * max(args.prompt, args.drafts + 1)
    model = Model(args.sequences, args.layers, args.prompt + (args.steps + 1) * (args.drafts + 1), rows, linear=args.linear)
    prompt = torch.randint(0, model.vocabulary, (args.sequences, args.prompt), dtype=torch.int32, device="cuda")
    accepted, tokens = run(model, prompt, args.drafts, args.steps)
    for s in range(args.sequences):
        row = [t for t in tokens[:, s].flatten().tolist() if t >= 0]
        print(f"sequence {s}: {len(row)} tokens, {int(accepted[:, s].sum())} of {args.drafts * args.steps} drafts accepted: {row[:12]} ...")
    model.release()


if __name__ == "__main__":
    main()
