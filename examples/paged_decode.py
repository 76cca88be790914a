"""Serving pages from a paged 8-bit KV cache: one attention layer decoding
several sequences at once.

    python examples/paged_decode.py [--seqs 8] [--prompt 6544] [--steps 64] [--fmt e4m3|i8]

A pool of pages serves sequences of different lengths.  Each prompt's keys and
values are rotated, quantized and stored by one append; then every step
embeds the sequences' last tokens, projects them, appends the new rows with
their rotation and attends over the cache, all captured once in a CUDA graph
(the lengths live on the device and move on inside it), and picks the next
tokens.  The weights are random; the sizes are those of one of the model's
layers (16 query heads, 8 KV heads, 64 wide).  Prints the picked tokens' first
few and the time of a step; exits with an error if a call reported one.
"""

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "falcon-ocr-cpu_b200"))
import fo_cuda as F  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE, VOCAB = 16, 8, 64, 64, 4096


def decode(seqs=8, prompt=6544, steps=64, fmt="e4m3", seed=0):
    """Returns the picked tokens [steps][seqs] and a step's microseconds."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    width = HEADS * DIM

    def weights(*shape):
        return (torch.randn(*shape, device="cuda", generator=g) * shape[0] ** -0.5).bfloat16()

    embed, project, head = weights(VOCAB, width) * VOCAB ** 0.5, weights(width, (HEADS + 2 * KV_HEADS) * DIM), weights(width, VOCAB)
    sinks = torch.randn(HEADS, device="cuda", generator=g)
    # Prompts between half of `prompt` and all of it; pages for them and for what is decoded, in any order.
    lens = [prompt - i * prompt // (2 * seqs) for i in range(seqs)]
    per_seq = -(-(prompt + steps + 1) // PAGE)
    pages = per_seq * seqs
    kind = torch.float8_e4m3fn if fmt == "e4m3" else torch.int8
    k_codes, v_codes = (torch.zeros(pages, KV_HEADS, PAGE, DIM, dtype=torch.int8, device="cuda").view(kind) for _ in range(2))
    k_scales, v_scales = (torch.zeros(pages, KV_HEADS, device="cuda") for _ in range(2))
    kv = F.PagedKv(k_codes, v_codes, k_scales, v_scales)
    page_table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).view(seqs, per_seq)
    rope = F.Rope(F.rope_table(torch.empty(prompt + steps + 1, DIM // 2, 2, device="cuda")))
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")

    # The prompts' keys and values, whatever computed them.
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    tokens = torch.randint(0, VOCAB, (start[-1],), device="cuda", generator=g)
    rows = (embed[tokens] @ project).view(-1, HEADS + 2 * KV_HEADS, DIM)
    F.paged_append(kv, F.PagedBatch(page_table, lengths, rows=max(lens),
                                    row_start=torch.tensor(start, dtype=torch.int32, device="cuda")),
                   rows[:, HEADS:HEADS + KV_HEADS], rows[:, HEADS + KV_HEADS:], rope=rope)

    batch = F.PagedBatch(page_table, lengths)
    last = tokens[torch.tensor(start[1:], device="cuda") - 1].clone()
    q, out = (torch.empty(seqs, HEADS, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def step():
        x = embed[last]
        row = (x @ project).view(seqs, HEADS + 2 * KV_HEADS, DIM)
        lengths.add_(1)
        F.paged_append(kv, batch, row[:, HEADS:HEADS + KV_HEADS], row[:, HEADS + KV_HEADS:], rope=rope, q=row[:, :HEADS],
                       q_out=q)
        F.paged_attention(kv, batch, q, out, sinks=sinks)
        last.copy_(((x + out.view(seqs, width)) @ head).argmax(-1))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once before the capture: the stream's context and scratch are made
        before = last.clone()
        step()
        last.copy_(before)
        lengths.sub_(1)  # its row is written again by the first step
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    picked = torch.empty(steps, seqs, dtype=last.dtype, device="cuda")
    with torch.cuda.stream(side):
        begin.record()
        for i in range(steps):
            graph.replay()
            picked[i].copy_(last)
        end.record()
        F.stream_context(0).synchronize()  # raises what a call reported on the device
    return picked.cpu(), begin.elapsed_time(end) * 1e3 / steps


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--seqs", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=6544)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--fmt", choices=("e4m3", "i8"), default="e4m3")
    args = ap.parse_args()
    picked, us = decode(args.seqs, args.prompt, args.steps, args.fmt)
    print("first tokens of the first sequences:", picked[:8].t()[:4].tolist())
    print("%.1f us a step, %.0f tokens/s" % (us, args.seqs / us * 1e6))
