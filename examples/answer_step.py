"""From PCM to a decoder block: the listener's soft tokens of each tick go through one
text-decoder block over a paged 8-bit K/V cache.

Three sessions hear different seeded audio; each 80 ms tick the tower yields two
soft tokens a session, the page directory plans where their keys and values go, the block
runs, and the plan is committed.  The second session leaves half way and its pages are
given back.  Runs on a GPU:  python examples/answer_step.py
"""
from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parents[1]


def load_package():
    name = "gemma4_omni_b200"
    if name not in sys.modules:
        folder = ROOT / "gemma-4-omni_b200"
        spec = importlib.util.spec_from_file_location(name, folder / "__init__.py", submodule_search_locations=[str(folder)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


def main(ticks: int = 12) -> dict:
    load_package()
    from gemma4_omni_b200 import _lib, runtime, synthetic
    from gemma4_omni_b200.config import SMALL
    from gemma4_omni_b200.decode_ops import PageDirectory
    from gemma4_omni_b200.decoder_block import DecoderBlock, DecoderConfig

    torch.cuda.set_device(0)
    n = 3
    tower = runtime.ListenerEngine(SMALL, max_sessions=8, weight_format=1, device="cuda:0")
    tower.load_weights(synthetic.synthetic_tower_weights(SMALL, 1), synthetic.synthetic_film_weights(SMALL, 2))
    block = DecoderBlock.synthetic(DecoderConfig(hidden=SMALL.text_hidden, heads=4, kv_heads=1, head_dim=64, ffn=1024), seed=3)
    pages = PageDirectory.create(sessions=8, max_pages=16, pages=64, page_tokens=16)
    cache = block.new_cache(pages.pages, pages.page_tokens)
    live, out = list(range(n)), None
    for tick in range(ticks):
        pcm = np.stack([synthetic.session_audio(4, s, 1, first_frame=tick, total_frames=ticks)[0] for s in live])
        rows = torch.tensor(live, dtype=torch.int32, device="cuda")
        frame = torch.full((len(live),), tick, dtype=torch.int64, device="cuda")
        tower.pack(rows, torch.zeros(len(live), dtype=torch.int64, device="cuda"), frame, frame.clone())
        soft = tower.step(torch.from_numpy(pcm).cuda(), kind=_lib.LB_INPUT_PCM)["soft"]
        tower.commit()
        tokens = soft.view(-1, SMALL.text_hidden)
        plan = pages.plan(rows, torch.full_like(rows, 2), max_tokens=tokens.shape[0])
        out = block.step(tokens, plan, cache, max_new=2)
        pages.commit(plan)
        if tick == ticks // 2:  # a session leaves
            gone = live.pop(1)
            tower.reset_handle(gone)
            pages.release(torch.tensor([gone], dtype=torch.int32, device="cuda"))
    status = {"tower": tower.status(), "cache": cache.status(), "pages": pages.status(), "plan": plan.status()}
    lengths = pages.lengths.tolist()
    tower.close()
    return {"out": out, "lengths": lengths, "status": status}


if __name__ == "__main__":
    result = main()
    print("tokens held per session:", result["lengths"], "status:", result["status"], "output:", tuple(result["out"].shape))
