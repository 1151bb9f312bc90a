"""The client's calls around a model whose head and embedding are two tables, with norms before and after (RWKV-7)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_two_tables_and_their_norms():
    """The input norm is folded into the embedding's table, the output norm is taken in float64 before the head's.  Rows are the
    table's to the bit, and each tick's greedy tokens the float64 model's on the same two tables."""
    import fhessm
    from fhessm import client
    from fhessm.rwkv7 import RWKV7Shape, Sites, _ln, block_step, new_state, synthetic_weights
    sh = RWKV7Shape(n_layer=2, n_embd=128, head_size=64, d_decay=16, d_aaa=16, d_mv=16, d_gate=16, dim_ffn=256, vocab_size=515)
    w, sites, lanes = synthetic_weights(sh), Sites(), 12
    folded = _ln(sites, "blocks.0.ln0", w["emb.weight"], w["blocks.0.ln0.weight"], w["blocks.0.ln0.bias"])
    emb = client.Q4Table.quantise(folded, group=32, device="cuda")
    head = client.Q4Table.quantise(w["head.weight"], group=64, device="cuda")
    rows64, head64 = (t.dequantise().double().cpu().numpy() for t in (emb, head))
    cx = fhessm.CryptoContext(logN=12, L=2, K=1, alpha=1, hw=64)
    state, tokens = new_state(sh, lanes), torch.arange(lanes, device="cuda") * 40
    for tick in range(3):
        rows = client.q4_rows(cx, tokens, emb)
        x = rows.double().cpu().numpy()
        assert np.array_equal(x, rows64[tokens.cpu().numpy()])
        v_first = None
        for i in range(sh.n_layer):
            x, v_first = block_step(sh, w, i, x, state[i], v_first, sites, ln0=False)
        normed = _ln(sites, "ln_out", x, w["ln_out.weight"], w["ln_out.bias"])
        held = torch.from_numpy(normed.astype(np.float32)).cuda()
        logits = client.q4_matvec(cx, held, head)
        tokens, lp = client.sample(cx, logits, torch.zeros(lanes, device="cuda"), temperature=0.0)
        exact = normed @ head64.T
        # x's rounding to float32, its 22 bits, and 128 sums
        tol = (2.0 ** -24 + 2.0 ** -22 + 136 * 2.0 ** -24) * (np.abs(normed) @ np.abs(head64).T)
        assert (np.abs(logits.double().cpu().numpy() - exact) <= tol).all()
        pick = exact[np.arange(lanes), tokens.cpu().numpy()]
        assert (pick >= exact.max(1) - 2 * tol.max(1)).all() and (lp == 0).all()
    cx.sync()
    cx.close()
