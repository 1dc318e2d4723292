"""How the attention with groups lays a step out, restated: which kernel a
group's prefix goes to, and the runs of tiles its workgroups get. bytes() is the
workspace that follows from it, which tests compare with the library's: a rule
that changes there makes the restatement fail, not the cases that rely on it."""
from types import SimpleNamespace

CUS, TILE, WIDE_TILE, WIDE_PAIRS, WIDE_WORK = 256, 128, 64, 48, 5 * 2.0 ** 28


def up(a, b):
    return -(-a // b)


def layout(kv_heads, hd, page, requests, rows, width, n_groups, q_heads, window=False):
    s = SimpleNamespace()
    group = q_heads // kv_heads
    pairs = rows * group
    some = max(1, min(requests, rows))
    s.ro = 1 if pairs <= 16 * some else 2
    per = pairs // max(1, min(n_groups, some))
    s.rp = max(s.ro, 1 if per <= 16 else 2)
    tokens = max(1, width * page)
    many = pairs * kv_heads * tokens * hd >= WIDE_WORK and per >= WIDE_PAIRS
    s.np = 0 if n_groups == 0 or window or not many else 2 if per <= 64 else 4
    if s.np == 4 and per > 128 and (
            (pairs // 256 + n_groups) * kv_heads * (tokens // WIDE_TILE) >= 12 * CUS):
        s.np = 8
    s.own_units = (pairs // (16 * s.ro) + some) * kv_heads
    s.prefix_units = (pairs // (16 * s.rp) + n_groups) * kv_heads if n_groups else 0
    s.wide_units = (pairs // (32 * s.np) + n_groups) * kv_heads if s.np else 0
    s.runs = min((s.own_units + s.prefix_units) * up(tokens, TILE), 2 * CUS)
    s.wide_runs = min(s.wide_units * up(tokens, WIDE_TILE), CUS)
    rows_of_parts = (2 * s.runs * 16 * s.rp + s.prefix_units * 16 * s.rp + s.own_units * 16 * s.ro
                     + 2 * s.wide_runs * 32 * s.np + s.wide_units * 32 * s.np)
    at = 16 + 32 * n_groups + up(4 * requests, 16) * 16 + 2 * up(4 * n_groups, 16) * 16
    at += 16 * (s.prefix_units + s.own_units + s.wide_units) + up(rows_of_parts * 8, 16) * 16
    s.bytes = at + rows_of_parts * hd * 4
    return s


def wide_runs(s, kv_heads, groups):
    """The runs of the kernel for many pairs: per workgroup its tiles as (group,
    unit, tile). groups: (pairs, tokens that it does) of each."""
    tiles = []
    for g, (pairs, done) in enumerate(groups):
        if done < WIDE_TILE or not pairs:
            continue
        for u in range(up(pairs, 32 * s.np) * kv_heads):
            tiles += [(g, u, t) for t in range(done // WIDE_TILE)]
    n = min(s.wide_runs, len(tiles))
    return [tiles[len(tiles) * i // n:len(tiles) * (i + 1) // n] for i in range(n)]
