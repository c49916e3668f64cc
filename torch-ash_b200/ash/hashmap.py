"""HashMap and HashSet containers over ASHEngine (API of ash/hashmap.py)."""
from typing import Dict, List, Optional, Union

import torch

from . import core
from .core import ASHEngine, ASHModule
from .quant import FORMATS, QuantizedRows, VALUE_TYPES, check_format, dequantize_rows

Values = Union[torch.Tensor, List[torch.Tensor], Dict[str, torch.Tensor]]


def _value_names(value_dims) -> Dict[str, int]:
    """Naming rule of ash/hashmap.py:24-37: int -> "default", list -> "default_i", dict as given."""
    if isinstance(value_dims, int):
        return {"default": value_dims}
    if isinstance(value_dims, list):
        return {f"default_{i}": d for i, d in enumerate(value_dims)}
    if isinstance(value_dims, dict):
        return dict(value_dims)
    raise ValueError("value_dims must be int, list or dict")


def _value_formats(value_formats, value_dims) -> Dict[str, str]:
    """{name: format} of the values kept in 8 bits; declared as the value_dims are, or one format for all."""
    names = _value_names(value_dims)
    if value_formats is None:
        return {}
    if isinstance(value_formats, str):
        given = {name: value_formats for name in names}
    elif isinstance(value_formats, list) and isinstance(value_dims, list) and len(value_formats) == len(value_dims):
        given = dict(zip(names, value_formats))
    elif isinstance(value_formats, dict) and isinstance(value_dims, dict) and value_formats.keys() <= names.keys():
        given = value_formats
    else:
        raise ValueError("value_formats must be a format, or formats in the form of value_dims")
    formats = {name: check_format(f) for name, f in given.items() if f is not None}
    for name in formats:
        if names[name] < 1:
            raise ValueError(f"value {name!r}: a row of at least one value is wanted")
        if name + "_scale" in names:
            raise ValueError(f"value {name!r} is kept with its scales: the name {name + '_scale'!r} is taken")
    return formats


class HashMap(ASHModule):
    """Hash map with values stored in registered buffers of ``capacity`` rows.

    ``value_formats`` (not in the reference): values kept in 8 bits a number with one float32 scale a row, ``"e4m3"`` or
    ``"int8"`` -- one format for all values, or given in the form of ``value_dims`` with None for those kept as they are.
    ``insert`` quantises the rows of new keys as it writes them (float32, float16 or bfloat16), ``find`` and ``items`` give
    what they read back as.  The buffers are ``<name>`` (the codes) and ``<name>_scale``; ``ash.quant`` has the rules.
    """

    def __init__(self, key_dim: int, value_dims: Union[int, List[int], Dict[str, int]], capacity: int,
                 device: Union[str, torch.device] = torch.device("cpu"),
                 value_formats: Union[None, str, List[Optional[str]], Dict[str, Optional[str]]] = None):
        super().__init__()
        self.value_formats = _value_formats(value_formats, value_dims)
        if self.value_formats and not hasattr(core.backend.HashMap, "insert_rows"):
            raise RuntimeError("values in 8 bits need the CUDA library")
        self.engine = ASHEngine(key_dim, capacity, device)
        self.value_dims = value_dims
        self.values = {}
        self._set_values(self._new_values(capacity))

    def _new_values(self, capacity: int) -> Dict[str, torch.Tensor]:
        """Zeroed buffers by name, those of scales among them."""
        values = {}
        for name, d in _value_names(self.value_dims).items():
            dtype = FORMATS[self.value_formats[name]] if name in self.value_formats else torch.get_default_dtype()
            values[name] = torch.zeros(capacity, d, dtype=dtype, device=self.engine.device)
            if name in self.value_formats:
                values[name + "_scale"] = torch.zeros(capacity, dtype=torch.float32, device=self.engine.device)
        return values

    def _set_values(self, new_values: Dict[str, torch.Tensor]) -> None:
        for name in self.values:
            delattr(self, name)
        self.values = new_values
        for name, v in new_values.items():
            self.register_buffer(name, v)

    def _apply(self, fn, recurse=True):
        """half(), double() and the like are about numbers: codes and scales keep their types, and go on being the buffers that
        the map writes."""
        kept = {n: self.values[n] for name in self.value_formats for n in (name, name + "_scale")}
        super()._apply(fn, recurse)
        for name, v in kept.items():
            if self._buffers[name] is not v:
                self._buffers[name] = self.values[name] = v.to(self._buffers[name].device)
        return self

    def _rows(self, name: str) -> QuantizedRows:
        return QuantizedRows(self.values[name], self.values[name + "_scale"])

    def _as_dict(self, values: Values) -> Dict[str, torch.Tensor]:
        if isinstance(values, torch.Tensor):
            assert isinstance(self.value_dims, int)
            return {"default": values}
        if isinstance(values, list):
            assert isinstance(self.value_dims, list)
            return {f"default_{i}": v for i, v in enumerate(values)}
        if isinstance(values, dict):
            assert isinstance(self.value_dims, dict)
            return values
        raise ValueError("values must be Tensor, list, or dict")

    def reinterpret_value_dict(self, values: Dict[str, torch.Tensor]) -> Values:
        """Give values back in the form ``value_dims`` was declared in."""
        if isinstance(self.value_dims, int):
            return values["default"]
        if isinstance(self.value_dims, list):
            return [values[f"default_{i}"] for i in range(len(self.value_dims))]
        if isinstance(self.value_dims, dict):
            return values
        raise ValueError("values must be Tensor, list, or dict")

    def _gather(self, indices: torch.Tensor) -> Values:
        return self.reinterpret_value_dict({
            name: dequantize_rows(self._rows(name), indices) if name in self.value_formats else self.values[name][indices]
            for name in _value_names(self.value_dims)})

    def insert(self, keys: torch.Tensor, values: Values) -> None:
        values = self._as_dict(values)
        if not self.value_formats:
            self.engine.insert(keys, values, self.values)
            return
        tables = {}
        for name, d in _value_names(self.value_dims).items():
            rows = values.get(name)
            if rows is None or rows.dim() != 2 or rows.shape[0] != keys.shape[0] or rows.shape[1] != d:
                raise ValueError(f"value {name!r} must be ({keys.shape[0]}, {d}), got "
                                 f"{None if rows is None else tuple(rows.shape)}")
            if name in self.value_formats and rows.dtype not in VALUE_TYPES:
                raise ValueError(f"value {name!r} must be float32, float16 or bfloat16, got {rows.dtype}")
            tables[name] = tuple(self._rows(name)) if name in self.value_formats else self.values[name]
        self.engine.insert_rows(keys, values, tables)

    def find(self, keys: torch.Tensor, return_indices: bool = True, return_values: bool = False,
             value_dtype: torch.dtype = torch.float32):
        """(masks[, indices][, values]) -- masks first, as ash/hashmap.py:72-95.

        Values kept in 8 bits come as ``value_dtype`` (float32, float16 or bfloat16), zeros for absent keys; the others
        have the row of index 0 there, as indexing with the indices of absent keys does."""
        assert return_indices or return_values, "Must return at least one of indices or values"
        if return_values and self.value_formats:
            if value_dtype not in VALUE_TYPES:
                raise ValueError(f"value_dtype must be float32, float16 or bfloat16, got {value_dtype}")
            kept = {name: tuple(self._rows(name)) for name in self.value_formats}
            names = _value_names(self.value_dims)
            indices, masks, values = self.engine.find_rows(keys, kept, value_dtype, return_indices or len(kept) < len(names))
            values = {name: values[name] if name in kept else self.values[name][indices] for name in names}
        elif return_values:
            indices, masks, values = self.engine.find_values(keys, self.values)
        else:
            indices, masks = self.engine.find(keys)
        ans = (masks,)
        if return_indices:
            ans += (indices,)
        if return_values:
            ans += (self.reinterpret_value_dict(values),)
        return ans

    def erase(self, keys: torch.Tensor) -> None:
        self.engine.erase(keys)

    def clear(self) -> None:
        for name, v in self.values.items():
            # codes as bytes, their scales beside them: a code that is NaN reads as NaN whatever its scale is
            (v.view(torch.uint8) if name in self.value_formats else v).zero_()
        self.engine.clear()

    def size(self) -> int:
        return self.engine.size()

    def resize(self, new_capacity: int) -> None:
        new_values = {
            name: torch.zeros(new_capacity, *v.shape[1:], dtype=v.dtype, device=self.engine.device)
            for name, v in self.values.items()
        }
        # codes move as bytes: not every operation knows their type
        as_bytes = lambda values: {name: v.view(torch.uint8) if name in self.value_formats else v for name, v in values.items()}
        self.engine.resize(new_capacity, as_bytes(self.values), as_bytes(new_values))
        self._set_values(new_values)

    def keys(self) -> torch.Tensor:
        return self.engine.keys()

    def items(self, return_indices: bool = True, return_values: bool = False):
        """(keys[, indices][, values]) of the active entries (ash/hashmap.py:129-150)."""
        assert return_indices or return_values, "Must return at least one of indices or values"
        active_keys, active_indices = self.engine.items()
        ans = (active_keys,)
        if return_indices:
            ans += (active_indices,)
        if return_values:
            ans += (self._gather(active_indices),)
        return ans


class HashSet(ASHModule):
    """Hash set: keys only (ash/hashmap.py:153-178)."""

    def __init__(self, key_dim: int, capacity: int, device: Union[str, torch.device]):
        super().__init__()
        self.engine = ASHEngine(key_dim, capacity, device)

    def insert(self, keys: torch.Tensor) -> None:
        self.engine.insert_keys(keys)

    def find(self, keys: torch.Tensor) -> torch.Tensor:
        return self.engine.contains(keys)

    def erase(self, keys: torch.Tensor) -> None:
        self.engine.erase(keys)

    def clear(self) -> None:
        self.engine.clear()

    def size(self) -> int:
        return self.engine.size()

    def resize(self, new_capacity: int) -> None:
        self.engine.resize(new_capacity)

    def keys(self) -> torch.Tensor:
        return self.engine.keys()
