"""Times of attention over whole caches, of rotary positions and of a decoder's steps with both (no counterpart in the reference,
whose dense mode is batch 1: engine.py:74-81).

    prompts   every token of a prompt over those before it (pages), torch's scaled_dot_product_attention beside
    pieces    the last N tokens of longer sequences; short runs of tokens; many sets of one query
    rope      rows turned, with turned parts that are whole 16-byte pieces and others
    steps     captured decode steps of the 12-layer, width-768 model with random weights: seg and dense, learned and rotary

Each time is the median over spans of some milliseconds that launch one graph again and again, which makes the call on three
sets of inputs in turn: microseconds a call (steps: milliseconds a replay).

Run: python -m treeattn_amd.bench_whole_cache [prompts] [pieces] [rope] [steps]
"""
import sys

import torch
import torch.nn.functional as F

from . import kernels as K
from . import positions
from .config import Config
from .engine import Decoder, decode_nsplit_dense, weights_from_ours
from .model import GPT

F32, BF16 = torch.float32, torch.bfloat16

# (sequences, heads, tokens, head size, type, rows a page)
PROMPTS = [(2, 12, 8192, 64, BF16, 64), (8, 12, 2048, 64, BF16, 64), (2, 8, 4096, 128, BF16, 64), (2, 12, 8192, 32, BF16, 64),
           (4, 12, 1024, 64, BF16, 64), (1, 12, 1024, 64, BF16, 64), (1, 12, 512, 64, BF16, 64), (2, 12, 1024, 64, BF16, 8),
           (2, 12, 1024, 64, F32, 64), (2, 12, 1024, 64, F32, 8)]
# (sequences, heads, tokens, positions, head size, type, rows a page)
PIECES = [(2, 12, 256, 8000, 64, BF16, 64), (1, 12, 256, 30000, 64, BF16, 64), (1, 8, 256, 8000, 128, BF16, 64),
          (4, 12, 64, 4000, 64, BF16, 64), (32, 12, 16, 1000, 64, BF16, 64), (64, 12, 8, 700, 64, BF16, 64),
          (8, 12, 5, 2500, 64, F32, 8), (8, 12, 1, 16000, 64, BF16, 64), (12, 12, 1, 16000, 64, BF16, 64),
          (32, 12, 1, 32768, 128, BF16, 64), (32, 12, 1, 32768, 32, BF16, 64), (32, 12, 1, 32768, 16, BF16, 64),
          (32, 12, 1, 32768, 64, BF16, 16), (32, 12, 1, 32768, 64, BF16, 2), (32, 12, 1, 500, 64, BF16, 64)]
# (sequences, heads, tokens, head size, turned elements, type)
ROPES = [(8, 24, 8191, 64, 64, BF16), (8, 24, 8191, 64, 24, BF16), (8, 24, 8191, 64, 20, BF16), (8, 24, 8191, 80, 20, BF16)]
# (sequences, tokens, positions)
STEPS = [(32, 32768, 65536), (32, 8192, 65536), (1, 131072, 262144), (1, 8192, 262144)]


def timed(calls, spans=9):
    """Microseconds a call, from HIP events around spans of some milliseconds of a graph of all calls."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for f in calls:
            f()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for f in calls:
            f()

    def span(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            g.replay()
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b) / n
    span(2)
    n = max(1, int(8.0 / span(3)))
    return sorted(span(n) for _ in range(spans))[spans // 2] * 1000 / len(calls)


def attention(B, H, N, T, D, dtype, leaf):
    """Calls of dense_attn on three caches: the last N tokens of B sequences of T."""
    calls = []
    ns = decode_nsplit_dense(B, H, N, T, D)
    for _ in range(3):
        nb = (T + leaf - 1) // leaf
        pool = torch.empty(B * H * nb, 2, leaf, D, device='cuda', dtype=dtype).normal_()
        table = torch.randperm(B * H * nb, device='cuda').to(torch.int32).view(B, H, nb)
        cache = K.PagedCache(pool, table, T)
        q = torch.randn(B, H, N, D, device='cuda').to(dtype)
        tq = torch.arange(T - N, T, device='cuda', dtype=torch.int32)
        ws, out = K.dense_attn_workspace(B, H, N, D, ns, 'cuda', H), torch.empty_like(q)
        calls.append(lambda q=q, c=cache, tq=tq, ws=ws, out=out: K.dense_attn(q, c, None, tq, out=out, nsplit=ns, ws=ws))
    return calls


def name_of(dtype):
    return str(dtype).split('.')[1]


def prompts():
    for B, H, N, D, dtype, leaf in PROMPTS:
        t = timed(attention(B, H, N, N, D, dtype, leaf))
        q, k, v = (torch.randn(B, H, N, D, device='cuda').to(dtype) for _ in range(3))
        ref = timed([lambda: F.scaled_dot_product_attention(q, k, v, is_causal=True)])
        flops = 4 * B * H * D * (N * (N + 1) / 2)
        print('prompt   %2d x %d heads of %3d x %5d tokens, %s, pages of %2d: %7.1f us, %5.0f TFLOP/s (torch %.1f us)'
              % (B, H, D, N, name_of(dtype), leaf, t, flops / t / 1e6, ref), flush=True)


def pieces():
    for B, H, N, T, D, dtype, leaf in PIECES:
        t = timed(attention(B, H, N, T, D, dtype, leaf))
        size = 2 * B * H * T * D * torch.finfo(dtype).bits // 8
        print('piece    %2d x %d heads of %3d x %3d tokens, the last of %5d, %s, pages of %2d: %6.1f us, %.2f TB/s of K and V'
              % (B, H, D, N, T, name_of(dtype), leaf, t, size / t / 1e6), flush=True)


def rope():
    for B, H, T, D, rot, dtype in ROPES:
        r = K.Rope(positions.rope_frequencies(rot)[0], 'cuda')
        pos = torch.arange(T, device='cuda', dtype=torch.int32)
        xs = [torch.randn(B, H, T, D, device='cuda').to(dtype) for _ in range(3)]
        t = timed([lambda x=x: K.rope(x, pos, r, out=x) for x in xs])
        size = 2 * xs[0].numel() * xs[0].element_size()
        print('rope     %2d x %d heads of %3d x %5d tokens, %d turned, %s: %6.1f us, %.2f TB/s'
              % (B, H, D, T, rot, name_of(dtype), t, size / t / 1e6), flush=True)


def steps():
    H, C, V, layers = 12, 768, 50304, 12
    for B, T0, Tcap in STEPS:
        for mode in ('seg', 'dense'):
            for rotary in ('', 'half'):
                tree = dict(leaf=64, arity=2, wmax=32, beam=32) if B > 1 else dict(leaf=128, arity=4, wmax=64, beam=64)
                cfg = Config(vocab_size=V, seq_len=Tcap, n_layer=layers, n_head=H, n_embd=C, attn='seg', neighbors=False, local=3,
                             rope=rotary, **tree)
                torch.manual_seed(3)
                m = GPT(cfg)
                W = weights_from_ours({k: x.detach().to(BF16).cuda() for k, x in m.state_dict().items()}, cfg)
                dec = Decoder(W, layers, H, C, Tcap, mode, cfg, 'cuda', batch=B, max_tokens=T0 + 400, reserve_ahead=300,
                              paged=True)
                idx = torch.randint(0, V, (B, T0), generator=torch.Generator().manual_seed(3)).cuda()
                dec.capture(dec.prefill(idx, chunk=4 if B > 1 else None).argmax(-1), T0)
                times = []
                for _ in range(40):
                    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                    a.record()
                    for _ in range(5):
                        dec.replay()
                    b.record()
                    torch.cuda.synchronize()
                    times.append(a.elapsed_time(b) / 5)
                print('step     %2d sequences of %6d tokens, %-5s %-6s: %.3f ms' % (B, T0, mode, rotary and 'rotary',
                                                                                   sorted(times)[20]), flush=True)
                del dec, W, m
                torch.cuda.empty_cache()


def main():
    parts = dict(prompts=prompts, pieces=pieces, rope=rope, steps=steps)
    want = sys.argv[1:] or list(parts)
    if any(x not in parts for x in want):
        raise SystemExit(__doc__)
    if not torch.cuda.is_available():
        raise SystemExit('bench_whole_cache needs a GPU')
    for x in want:
        parts[x]()


if __name__ == '__main__':
    main()
