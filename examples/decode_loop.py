"""A decode loop of the small encrypted model with a 4-bit tied table: the server's tick on ciphertexts, and the client's
token step (head, choice, next row) on the same GPU.

    python examples/decode_loop.py [--ticks 3] [--temperature 0.8] [--top-k 40] [--top-p 0.95]

Needs a GPU and the built library (python __graft_entry__.py).  The weights are synthetic: the tokens mean nothing, the
path is the one of a trained model.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "fhe-ssm_b200"))

import fhessm
from fhessm.client import Q4Table, TokenHead
from fhessm.model import EncryptedModel, ModelConfig, calibrate_seeds, pack_lanes, synthetic_weights, unpack_lanes


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--ticks", type=int, default=3)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=40)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()

    cfg = ModelConfig(d=48, dff=128, n_layer=2, vocab=512, D=64, b1=8)
    weights = synthetic_weights(cfg, seed=5)
    table = Q4Table.quantise(weights["emb"], group=32)       # once; the model is calibrated on what the table holds
    weights["emb"] = table.dequantise().double().numpy()
    seeds = calibrate_seeds(cfg, weights, steps=3, lanes=128)

    cx = fhessm.CryptoContext(logN=13, L=28, K=4, alpha=4, hw=192, boot_primes=14)
    cx.KeyGen(seed=9)
    cx.EvalBootstrapSetup(24.0, 59)
    model = EncryptedModel(cx, cfg, weights, seeds)
    model.keygen()
    head = TokenHead(cx, table)

    lanes = 2 * cx.slots // cfg.D
    rng = torch.Generator(device=head.table.weight.device).manual_seed(a.seed)
    tokens = torch.randint(0, cfg.vocab, (lanes,), generator=rng, device=rng.device)
    rows = head.embed(tokens)
    for tick in range(a.ticks):
        ct = cx.Encrypt(cx.MakeCKKSPackedPlaintext(pack_lanes(rows.double().cpu().numpy(), cfg.D, cx.slots)))
        normed = unpack_lanes(cx.Decrypt(model.step(ct)), cfg.D, lanes, cfg.d)
        u = torch.rand(lanes, generator=rng, device=rng.device)
        tokens, logprob, rows = head.step(normed, u, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p)
        torch.cuda.current_stream().synchronize()
        cx.sync()                                            # raises if the tick lost anything to a wait that ran out
        print(f"tick {tick}: {lanes} conversations, mean log-probability {logprob.mean().item():.3f}, "
              f"first tokens {tokens[:8].tolist()}")
    cx.close()


if __name__ == "__main__":
    main()
