"""Batches of texts for the attention's tests, and the formulas in 64 bits."""

import math

import numpy as np

from operator_helpers import FLOOR, UNIT, from_bits, kind_code, strided, to_bits

STEP = 2.0 ** -23  # one float32 addition of the matrix cores, whose rounding need not be to nearest


class Batch:
    """q_lens and k_lens: rows that count of each text (k_lens None: q_lens, the same rows). lead: rows of no text before
    the first; room: rows of a padded text (lengths are passed), None: packed. Rows that do not count hold NaN."""

    def __init__(self, capi, kind, q_lens, *, k_lens=None, heads=2, kv_heads=None, head_dim=32, mask="full", prefix=None,
                 last=False, cap=0.0, bias=None, far=0, scale=None, lead=0, tail=0, room=None, pad=0, shift=0, spread=1.0, seed=1):
        rng = np.random.default_rng(seed)
        self.capi, self.kind, self.heads, self.head_dim = capi, kind, heads, head_dim
        self.kv_heads = kv_heads or heads
        self.q_lens, self.k_lens = list(q_lens), list(q_lens if k_lens is None else k_lens)
        self.mask, self.last, self.cap, self.bias, self.far = mask, last, cap, bias, far
        self.scale = head_dim ** -0.5 if scale is None else scale
        self.texts = len(self.q_lens)
        self.prefix = [int(p) for p in prefix] if prefix is not None else [0] * self.texts
        apart = k_lens is not None
        self.q_starts, self.q_rows = self._layout(self.q_lens, lead, tail, None if apart else room)
        self.k_starts, self.k_rows = self._layout(self.k_lens, lead, tail, room) if apart else (self.q_starts, self.q_rows)
        self.owners = []

        def rows(count, starts, lens, n):
            values = np.full((count, n * head_dim), np.nan)
            for start, length in zip(starts, lens):
                values[start:start + length] = spread * rng.standard_normal((length, n * head_dim))
            owner, address, stride, stored = strided(capi, values, kind, pad, shift)
            self.owners.append(owner)
            return address, stride, stored

        q, self.q_stride, self.q = rows(self.q_rows, self.q_starts, self.q_lens, heads)
        k, self.k_stride, self.k = rows(self.k_rows, self.k_starts, self.k_lens, self.kv_heads)
        v, self.v_stride, self.v = rows(self.k_rows, self.k_starts, self.k_lens, self.kv_heads)
        self.slopes = np.float32(2.0) ** (-np.arange(1, heads + 1, dtype=np.float32)) if bias == "slopes" else None
        self.table = None
        if bias == "table":
            stored = to_bits(rng.standard_normal((heads, 2 * far + 1)), kind)
            self.table = from_bits(stored, kind)
            table = self._keep(stored)

        def offsets(starts, lens):
            return self._keep(np.array(list(starts) + [starts[-1] + lens[-1] if lens else lead], np.int64))

        padded = room is not None
        lengths = (self._keep(np.array(self.k_lens, np.int32)) if padded else None)
        self.desc = capi.attention_desc(
            q, k, v, self.texts, self.q_rows, self.k_rows, heads, head_dim, kind_code(capi, kind), kv_heads=self.kv_heads,
            q_offsets=None if padded and not apart else offsets(self.q_starts, self.q_lens),
            k_offsets=None if padded else offsets(self.k_starts, self.k_lens),
            q_lengths=lengths if padded and not apart else None, k_lengths=lengths,
            q_align=capi.ATTENTION_LAST if last else capi.ATTENTION_FIRST, causal=mask != "full",
            prefix_lengths=self._keep(np.array(self.prefix, np.int32)) if mask == "prefix" else None, scale=self.scale,
            cap=cap, slopes=self._keep(self.slopes) if bias == "slopes" else None,
            distance_bias=table if bias == "table" else None, max_distance=far, q_stride=self.q_stride,
            k_stride=self.k_stride, v_stride=self.v_stride)

    def _keep(self, host):
        array = self.capi.DeviceArray.from_host(host)
        self.owners.append(array)
        return array

    @staticmethod
    def _layout(lens, lead, tail, room):
        if room is not None:
            return [t * room for t in range(len(lens))], len(lens) * room
        starts = [lead + sum(lens[:t]) for t in range(len(lens))]
        return starts, lead + sum(lens) + tail

    def of_text(self, t):
        """q, k, v of one text [heads, rows, head_dim] (keys repeated for their query heads), positions, keys seen."""
        q = self.q[self.q_starts[t]:][:self.q_lens[t]].reshape(-1, self.heads, self.head_dim).transpose(1, 0, 2)
        k, v = (np.repeat(x[self.k_starts[t]:][:self.k_lens[t]].reshape(-1, self.kv_heads, self.head_dim).transpose(1, 0, 2),
                          self.heads // self.kv_heads, axis=0) for x in (self.k, self.v))
        place = np.arange(self.q_lens[t]) + (self.k_lens[t] - self.q_lens[t] if self.last else 0)
        distance = np.arange(self.k_lens[t])[None, :] - place[:, None]
        seen = np.ones_like(distance, dtype=bool)
        if self.mask != "full":
            seen = (distance <= 0) | (np.arange(self.k_lens[t])[None, :] < (self.prefix[t] if self.mask == "prefix" else 0))
        return q, k, v, distance, seen

    def scores(self, q, k, distance, table=None):
        """Scores before the masks, the cap's derivative, and the scores' errors in float32 (see softmax_error)."""
        raw = q @ k.transpose(0, 2, 1) * self.scale
        error = (self.head_dim + 4) * STEP * abs(self.scale) * (np.abs(q) @ np.abs(k).transpose(0, 2, 1))
        slope = np.ones_like(raw)
        if self.cap:
            t = np.tanh(raw / self.cap)
            raw, slope = self.cap * t, 1.0 - t * t
            error = error + 2.0 ** -20 * self.cap  # the tangent's own error
        if self.slopes is not None:
            raw = raw - self.slopes.astype(np.float64)[:, None, None] * np.abs(distance)
        table = self.table if table is None else table
        if table is not None:
            raw = raw + table[:, np.clip(distance, -self.far, self.far) + self.far]
        # factors of base 2, biases and the difference from the maximum, a few roundings of the values they have
        size = np.abs(raw)
        error = error + 2.0 ** -21 * (size + (size.max(2, keepdims=True) if size.shape[2] else 0.0))
        return raw, slope, error

    def softmax(self, scores, seen):
        masked = np.where(seen, scores, -np.inf)
        top = masked.max(2, keepdims=True, initial=-np.inf)
        p = np.where(seen, np.exp(masked - np.where(np.isfinite(top), top, 0.0)), 0.0)
        total = p.sum(2, keepdims=True)
        with np.errstate(divide="ignore"):
            lse = (np.where(np.isfinite(top), top, 0.0) + np.log(total))[..., 0]
        return p / np.where(total > 0, total, 1.0), np.where(total[..., 0] > 0, lse, -np.inf)

    def forward(self):
        """Rows [q_rows, heads * head_dim] (NaN: not written), their tolerance, lse [q_rows, heads] and its tolerance."""
        out = np.full((self.q_rows, self.heads * self.head_dim), np.nan)
        tolerance, lse, lse_tolerance = np.zeros_like(out), np.full((self.q_rows, self.heads), np.nan), np.zeros((self.q_rows, self.heads))
        for t in range(self.texts):
            q, k, v, distance, seen = self.of_text(t)
            scores, _, error = self.scores(q, k, distance)
            p, text_lse = self.softmax(scores, seen)
            n = self.k_lens[t]
            worst = np.where(seen, error, 0.0).max(2, keepdims=True, initial=0.0)
            mass = p @ np.abs(v)
            # each exponential's and the sum's errors, its rounding for the product with v (below the smallest normal
            # number by itself; the sum is at least 1), the sums over the keys
            own = (2.02 * worst + (0 if self.kind == "f32" else UNIT[self.kind]) + (n + 8) * STEP) * mass
            own = own + FLOOR[self.kind] * np.abs(v).sum(1, keepdims=True)
            text_out = p @ v
            own = own + UNIT[self.kind] * (np.abs(text_out) + own) + FLOOR[self.kind]
            rows = slice(self.q_starts[t], self.q_starts[t] + self.q_lens[t])
            out[rows] = text_out.transpose(1, 0, 2).reshape(self.q_lens[t], out.shape[1])
            tolerance[rows] = own.transpose(1, 0, 2).reshape(self.q_lens[t], out.shape[1])
            lse[rows] = text_lse.T
            finite = np.where(np.isfinite(text_lse), np.abs(text_lse), 0.0)
            lse_tolerance[rows] = (1.01 * worst[..., 0] + (n + 8) * STEP + 2.0 ** -21 * (finite + 1.0)).T
        return out, tolerance, lse, lse_tolerance

    def gradient(self, g, out_stored):
        """name -> (gradient, its tolerance), NaN in rows of no text and zeros in padding rows, from the output's gradient
        g and the output as it is handed to the kernel."""
        width = self.heads * self.head_dim
        shapes = dict(q=(self.q_rows, width), k=self.k.shape, v=self.v.shape)
        value = {n: np.full(s, np.nan) for n, s in shapes.items()}
        error = {n: np.zeros(s) for n, s in shapes.items()}
        unit, floor = UNIT[self.kind], FLOOR[self.kind]
        inner, inner_floor = (0.0, 0.0) if self.kind == "f32" else (unit, floor)
        bins = 2 * self.far + 1
        table, table_error = np.zeros((self.heads, bins)), np.zeros((self.heads, bins))
        ratio = self.heads // self.kv_heads
        for t in range(self.texts):
            q, k, v, distance, seen = self.of_text(t)
            nq, nk = self.q_lens[t], self.k_lens[t]
            rows = slice(self.q_starts[t], self.q_starts[t] + nq)
            keys = slice(self.k_starts[t], self.k_starts[t] + nk)
            dout = g[rows].reshape(nq, self.heads, self.head_dim).transpose(1, 0, 2)
            out = out_stored[rows].reshape(nq, self.heads, self.head_dim).transpose(1, 0, 2)
            scores, slope, s_error = self.scores(q, k, distance)
            p, lse = self.softmax(scores, seen)
            lse_size = np.where(np.isfinite(lse), np.abs(lse), 0.0)[..., None]
            p_error = p * (1.02 * (s_error + 2.0 ** -21 * (lse_size + 1.0)))
            dp = dout @ v.transpose(0, 2, 1)
            delta = (p * dp).sum(2, keepdims=True)
            dp_error = (self.head_dim + 2) * STEP * (np.abs(dout) @ np.abs(v).transpose(0, 2, 1))
            # the output's own rounding is in the kernel's delta
            exact_out = p @ v
            delta_error = ((np.abs(dout) * (np.abs(out - exact_out) + (self.head_dim + 2) * STEP * np.abs(out))).sum(2, keepdims=True))
            ds = p * (dp - delta)
            ds_error = p_error * np.abs(dp - delta) + (p + p_error) * (dp_error + delta_error) + 4 * STEP * np.abs(ds)
            dr = ds * slope
            dr_error = ds_error * slope + (2.0 ** -18 * np.abs(ds) if self.cap else 0.0)
            dr_error = dr_error + inner * (np.abs(dr) + dr_error) + inner_floor
            p_rounded = p_error + inner * (p + p_error) + inner_floor
            # masked places take no part
            dr_error, p_rounded, ds_error = (np.where(seen, e, 0.0) for e in (dr_error, p_rounded, ds_error))
            size = abs(self.scale)
            results = dict(q=(dr @ k * self.scale, size * (dr_error @ np.abs(k) + (nk + 6) * STEP * (np.abs(dr) + dr_error) @ np.abs(k))))
            turned = np.abs(dr).transpose(0, 2, 1) + dr_error.transpose(0, 2, 1)
            results["k"] = (dr.transpose(0, 2, 1) @ q * self.scale,
                            size * (dr_error.transpose(0, 2, 1) @ np.abs(q) + (nq * ratio + 6) * STEP * turned @ np.abs(q)))
            turned = p.transpose(0, 2, 1) + p_rounded.transpose(0, 2, 1)
            results["v"] = (p.transpose(0, 2, 1) @ dout,
                            p_rounded.transpose(0, 2, 1) @ np.abs(dout) + (nq * ratio + 6) * STEP * turned @ np.abs(dout))
            for name, (grad, own) in results.items():
                n = nq if name == "q" else nk
                if name != "q":  # summed over the heads of a key head
                    grad, own = (x.reshape(self.kv_heads, ratio, n, self.head_dim).sum(1) for x in (grad, own))
                own = own + unit * (np.abs(grad) + own) + floor
                where = rows if name == "q" else keys
                value[name][where] = grad.transpose(1, 0, 2).reshape(n, shapes[name][1])
                error[name][where] = own.transpose(1, 0, 2).reshape(n, shapes[name][1])
            if self.table is not None:
                at = (np.clip(distance, -self.far, self.far) + self.far).ravel()
                for i in range(self.heads):
                    np.add.at(table[i], at, ds[i].ravel())
                    np.add.at(table_error[i], at, (ds_error[i] + (nq + nk + 64) * STEP * np.abs(ds[i])).ravel())
        if self.table is not None:
            value["table"], error["table"] = table, table_error + unit * (np.abs(table) + table_error) + floor
        return {name: (value[name], error[name]) for name in value}
