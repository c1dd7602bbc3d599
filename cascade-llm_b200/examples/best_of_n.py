"""Best of n: n sampled continuations of one prompt, ranked by mean log probability
(of each token among those that temperature, top-k and top-p kept for it).

    python cascade-llm_b200/examples/best_of_n.py [--checkpoint DIR] [--n 8] [--new-tokens 32]

Without a checkpoint the weights are the seeded random ones of the benchmark and
the prompt is random ids. The prompt runs once; its pages are shared by the
continuations, which then decode together, one token each per step.
"""

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import layer_streaming as ls  # noqa: E402


class Config:
    hidden_size, intermediate_size, num_hidden_layers = 4096, 14336, 32
    num_attention_heads, num_key_value_heads, vocab_size = 32, 8, 128256
    rms_norm_eps = 1e-5
    rope_parameters = {
        "rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
        "original_max_position_embeddings": 8192, "rope_theta": 500000.0,
    }


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--checkpoint", help="directory with a Llama-3.1-8B checkpoint (safetensors)")
    parser.add_argument("--n", type=int, default=8)
    parser.add_argument("--prompt-tokens", type=int, default=512)
    parser.add_argument("--new-tokens", type=int, default=32)
    parser.add_argument("--temperature", type=float, default=0.8)
    parser.add_argument("--top-k", type=int, default=50)
    parser.add_argument("--top-p", type=float, default=0.95)
    parser.add_argument("--seed", type=int, default=0)
    args = parser.parse_args()

    device = torch.device("cuda:0")
    plan = ls.build_llama31_8b_plan("matrix_group")
    store = ls.create_weight_store(plan, "full_pinned")
    if args.checkpoint:
        store.load_checkpoint(args.checkpoint)
    else:
        store.fill_seeded(seed=0, device=device)
    resident = ls.ResidentDeviceArena(plan, store, device)
    runtime = ls.DoubleBufferRuntime(plan, store, resident, device, weights="hbm")
    executor = ls.Llama31DecodeExecutor(Config(), resident, max_length=args.prompt_tokens)

    length = args.prompt_tokens + args.new_tokens
    pages = -(-args.prompt_tokens // 16) + args.n * (-(-args.new_tokens // 16) + 1)
    decoder = ls.PagedBatchDecoder(executor, runtime, sequences=args.n, pages=pages, max_length=length)
    prompt = torch.randint(0, Config.vocab_size, (1, args.prompt_tokens),
                           generator=torch.Generator().manual_seed(args.seed)).to(device)
    generator = torch.Generator(device=device).manual_seed(args.seed)
    for attempt in ("first (captures the step)", "second"):
        torch.cuda.synchronize()
        started = time.perf_counter()
        tokens, logprobs = decoder.best_of(prompt, args.new_tokens, generator, args.temperature, args.top_k, args.top_p)
        torch.cuda.synchronize()
        seconds = time.perf_counter() - started
        print("{}: {} x {} tokens in {:.3f} s ({:.0f} tokens/s)".format(
            attempt, args.n, args.new_tokens, seconds, args.n * args.new_tokens / seconds))
    mean = logprobs.mean(1)
    for rank, i in enumerate(mean.argsort(descending=True).tolist()):
        print("{:2d}. continuation {} mean log probability {:.3f}: {} ...".format(
            rank + 1, i, float(mean[i]), tokens[i, :8].tolist()))


if __name__ == "__main__":
    main()
