// What the GEMM's epilogue needs to add low-rank adapters to its rows.
#pragma once

struct AdapterRows {
    const void* inner;          // bf16 [M][rank_pad], zero behind rank
    const void* up;             // bf16 [n_adapters][N][rank]
    const int* row_ids;         // adapter of rows_per_id rows each
    int rows_per_id, n_adapters, rank, rank_pad;
};
