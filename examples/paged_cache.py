"""A serving loop's cache, from prompt to archive: chunks of a prompt and single
tokens are appended and attended to, the attention that every token receives is
recorded, the cache is cut back to a budget when it outgrows it, and a finished
sequence's layers go through the codec.

    python examples/paged_cache.py [--tokens 4096] [--budget 2048] [--layers 2]

Keys, values and queries are random: the example shows the calls, not a model.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import kvforge_b200 as kvf  # noqa: E402

HEADS, QUERY_HEADS, DIM, PAGE = 8, 32, 128, 64
RECENT, SINKS = 256, 4


def step(cache, seqs, counts, layers, gen):
    """One forward step: counts[i] new tokens of sequence seqs[i] in every layer."""
    batch = cache.extend(seqs, counts, query_heads=QUERY_HEADS)
    rows = lambda heads: torch.randn((batch.tokens, heads, DIM), generator=gen, device="cuda").half()  # noqa: E731
    for layer in range(layers):
        cache.append(batch, rows(HEADS), rows(HEADS), layer)
        out = cache.attend(batch, rows(QUERY_HEADS), layer, decay=1.0)
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=4096, help="tokens of the longer prompt")
    ap.add_argument("--budget", type=int, default=2048, help="tokens a sequence may keep")
    ap.add_argument("--layers", type=int, default=2)
    args = ap.parse_args()
    gen = torch.Generator(device="cuda").manual_seed(0)

    # room for two sequences, and for the pages that an eviction moves to
    pages = 3 * (args.tokens // PAGE + 2) + args.budget // PAGE + 2
    cache = kvf.PagedKVCache(pages, HEADS, DIM, page_size=PAGE, num_layers=args.layers, dtype=torch.float16)
    a, b = cache.add(), cache.add()

    # prompts in chunks, the shorter one's tokens in the same batches
    left = [args.tokens, args.tokens // 3]
    while any(left):
        counts = [min(n, 1024) for n in left]
        step(cache, [a, b], counts, args.layers, gen)
        left = [n - c for n, c in zip(left, counts)]
    print(f"prompts: {cache.length(a)} and {cache.length(b)} tokens, {cache.free_pages} of {pages} pages free")

    # answers, token by token; what outgrows the budget is evicted by weight
    for _ in range(16):
        over = [s for s in (a, b) if cache.length(s) > args.budget + 64]
        if over:
            kept = cache.evict(over, args.budget, recent=RECENT, sinks=SINKS).kept
            print(f"evicted to {args.budget} tokens; layer 0, head 0 keeps {kept[0, 0, 0, :8].tolist()} ...")
        out = step(cache, [a, b], [1, 1], args.layers, gen)
    cache.sync()  # raises if a kernel gave up
    print(f"answers: {cache.length(a)} and {cache.length(b)} tokens, output {tuple(out.shape)}")

    # a finished sequence goes to the archive, layer by layer, and its pages are free again
    for layer in range(args.layers):
        c = kvf.compress(cache.gather(a, layer), "conservative")
        back = kvf.decompress(c)
        print(f"layer {layer}: {c!r}, restored {back.shape}")
    cache.free(a)
    print(f"{cache.free_pages} of {pages} pages free")


if __name__ == "__main__":
    main()
