"""From camera features to answers about one scene.

Camera features are pooled into a BEV map (lss_bev_pool_depth); the map's cells
and the cameras' pixels become the tokens of a scene, with positions (frame,
row, column).  An attention layer is trained one step on two scenes packed into
one row of tokens.  Then one scene's keys and values are computed once, and
several questions about it are answered token by token, each with a short cache
of its own.

    python examples/bev_tokens.py
"""
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))

from __graft_entry__ import load_package  # noqa: E402

CHANNELS, CELL = 80, 6  # of the map; cells a token covers each way


def scene_tokens(pkg, rig, context):
    """(tokens, positions) of one sample: the pooled map's patches, then the
    cameras' pixels.  context (cameras, C, fH, fW)."""
    from bevfusion_triton_amd import synthetic

    geom = synthetic.make_geometry(rig).to(context.device)
    pool = pkg.BevPoolTransform(rig.xbound, rig.ybound, rig.zbound).to(context.device)
    depth = torch.full((geom.shape[1], *geom.shape[2:5]), 1.0 / geom.shape[2],
                       device=context.device)
    bev = pool.bev_pool_depth(geom, depth, context)
    bev = torch.nn.functional.avg_pool2d(bev, CELL)  # (1, C, rows, columns)
    maps = [bev] + [c[None] for c in context]
    tokens = torch.cat([m[0].flatten(1).T for m in maps])
    positions = torch.cat([
        torch.cartesian_prod(torch.tensor([frame]), torch.arange(m.shape[2]),
                             torch.arange(m.shape[3])) for frame, m in enumerate(maps)])
    return tokens, positions.to(context.device)


def main(device='cuda:0', dtype=torch.bfloat16, questions=3, answer=5):
    pkg = load_package()
    from bevfusion_triton_amd import synthetic

    torch.manual_seed(0)
    rig = synthetic.CASES['tiny']
    cameras, (fh, fw) = 6, rig.feature
    layer = pkg.TokenAttention(CHANNELS, 8, 2, 64, (8, 12, 12), device=device, dtype=dtype)

    # one training step on two scenes of their own lengths, packed
    scenes = [scene_tokens(pkg, rig, torch.randn(cameras, CHANNELS, fh, fw, device=device))
              for _ in range(2)]
    scenes[1] = tuple(t[:-fh * fw] for t in scenes[1])  # a camera less
    x = torch.cat([t for t, _ in scenes]).to(dtype)
    positions = torch.cat([p for _, p in scenes])
    starts = torch.tensor([0, *(len(t) for t, _ in scenes)]).cumsum(0).to(device)
    loss = (layer(x, positions, starts) - x).float().square().mean()
    loss.backward()
    with torch.no_grad():
        for p in layer.parameters():
            p -= 0.1 * p.grad
    print(f'trained on {len(x)} tokens of {len(scenes)} scenes: loss {loss.item():.4f}')

    # questions about the first scene: its keys and values once for all
    tokens, places = scenes[0]
    prefix = layer.scene(tokens.to(dtype), places)
    cache_k = torch.zeros((questions, answer, 2, 64), device=device, dtype=dtype)
    cache_v, lengths = torch.zeros_like(cache_k), torch.zeros(questions, dtype=torch.int32,
                                                              device=device)
    token = torch.randn((questions, 1, CHANNELS), device=device, dtype=dtype)
    asked, given = [], []
    for i in range(answer):
        at = torch.full((questions, 1, 3), cameras + 1 + i, device=device)
        asked.append(token)
        token = token + layer.step(token, at, cache_k, cache_v, lengths, prefix)
        given.append(token)
    print(f'{questions} questions over a scene of {len(tokens)} tokens: '
          f'{answer} tokens each')
    return {'layer': layer, 'scene': (tokens.to(dtype), places), 'asked': torch.cat(asked, 1),
            'given': torch.cat(given, 1), 'first': cameras + 1, 'loss': loss.detach()}


if __name__ == '__main__':
    main()
