/*
 * libipus: C ABI of the MI355X (gfx950) backend for the ipu-stack hot path.
 *
 * This header is the drop-in boundary.  It replaces the roles that the
 * reference splits over four Rust crates:
 *   - ipu-runtime / ipu-driver (device open, host sessions, PCIe exchange):
 *       crates/ipu-runtime/src/lib.rs:17-47, crates/ipu-driver/src/lib.rs:1341-1600
 *     -> ipus_context_*, ipus_buffer_*, ipus_stream_sync, ipus_event_*
 *   - ipu-elf (compile + link, symbol lookup): crates/ipu-elf/src/lib.rs:86-170, 322
 *     -> kernels are compiled into this library; ipus_kernel_abi looks them up
 *   - ipu-target (ComputeStep emission: m2 = output, m3.. = inputs, then u32
 *     scalars): crates/ipu-target/src/program.rs:112-121,
 *     crates/ipu-target/src/emit.rs:514-551,
 *     crates/ipu-codegen/src/kernel.rs:14-16, 818-865
 *     -> ipus_launch(symbol, out, inputs, scalars)
 *   - the tile-kernel ABI registry and run validation:
 *     crates/ipu-codegen/src/kernel.rs:1215-1435 (tile_kernel_abi,
 *     validate_kernel_run) -> ipus_kernel_abi + the checks inside ipus_launch.
 *
 * Conventions (kernel.rs:14-16, crates/ipu-codegen/src/operator.rs:467-537):
 *   - The caller owns every buffer.  Kernels read inputs and write the output
 *     and allocate nothing.  A context holds 96 MiB of device memory of its
 *     own (32 MiB where there is no room for more) for launches that merge
 *     partial results (allocated with it, outside ipus_context_live_buffers).
 *   - Launches are ordered on the context's stream (replacing BSP phases).
 *     Threads may share a context: the launches of one call, of a session's run
 *     and of a capture stand together, whatever other threads enqueue.
 *   - Every call returns 0 on success or a negative IPUS_ERROR_* code;
 *     ipus_last_error() returns the message of the calling thread's last
 *     failure.  HIP runtime failures map to IPUS_ERROR_HIP_BASE - hipError_t.
 *   - Scalars are u32, as in the reference's PlannedKernelCall::arguments
 *     (kernel.rs:136-140).  f32 values travel as their bit patterns, as in
 *     AttentionScale::ValueBits (crates/ipu-codegen/src/graph.rs:147-165).
 */
#ifndef IPUS_H
#define IPUS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes (KernelAbiError, kernel.rs:140-162) ---- */
#define IPUS_OK 0
#define IPUS_ERROR_INVALID_ARGUMENT (-1)   /* RequirementMismatch / bad shape */
#define IPUS_ERROR_POINTER_ARITY (-2)      /* PointerArity { expected, actual } */
#define IPUS_ERROR_UNAVAILABLE (-3)        /* Unavailable(spec): no device kernel */
#define IPUS_ERROR_UNSUPPORTED_COUNT (-4)  /* UnsupportedElementCount */
#define IPUS_ERROR_UNKNOWN_SYMBOL (-5)     /* symbol not in the registry */
#define IPUS_ERROR_GRAPH (-6)              /* GraphError (graph.rs:221-245) */
#define IPUS_ERROR_BUILD (-7)              /* PackageBuildError (package.rs:48-78) */
#define IPUS_ERROR_NO_DEVICE (-8)
#define IPUS_ERROR_OUT_OF_MEMORY (-9)
/* A reference symbol that names an IPU tile codelet with no per-tile GPU
 * counterpart (the tile GEMM codelets, the staged-attention codelets): the
 * caller translates the whole operator to one launch instead.  The message
 * names the replacement symbol. */
#define IPUS_ERROR_TRANSLATED (-10)
#define IPUS_ERROR_HIP_BASE (-1000)        /* IPUS_ERROR_HIP_BASE - hipError_t */

/* Message of the calling thread's most recent failure ("" if none). */
const char *ipus_last_error(void);
/* Library version string. */
const char *ipus_version(void);

/* ---- context: one device, one stream (Runtime::open / HostSession) ---- */
typedef struct ipus_context ipus_context;

typedef struct ipus_device_info {
  char name[64];          /* e.g. "AMD Instinct MI355X"; where the runtime
                             reports none, the driver's sysfs product_name
                             of the device's PCI function */
  char arch[32];          /* gcnArchName, e.g. "gfx950:sramecc+:xnack-" */
  int compute_units;
  int clock_khz;
  int memory_clock_khz;
  int memory_bus_width;
  uint64_t global_memory_bytes;
  int lds_bytes_per_block;
} ipus_device_info;

int ipus_device_count(int *count);
int ipus_context_create(int device, ipus_context **out);
int ipus_context_destroy(ipus_context *context);
int ipus_context_device_info(ipus_context *context, ipus_device_info *info);
/* Stream handle (hipStream_t) of the context, for callers that interoperate
 * with other HIP code.  Launches through this library go to this stream. */
int ipus_context_stream(ipus_context *context, void **stream);

/* ---- buffers: replace SRAM placement, host exchange and FillZero ---- */
int ipus_buffer_alloc(ipus_context *context, size_t bytes, void **device_pointer);
int ipus_buffer_free(ipus_context *context, void *device_pointer);
/* Synchronous host <-> device copies (complete before returning). */
int ipus_buffer_upload(ipus_context *context, void *device_dst, const void *host_src,
                       size_t bytes);
int ipus_buffer_download(ipus_context *context, void *host_dst, const void *device_src,
                         size_t bytes);
/* Buffers allocated through the context and not yet freed (count, bytes).
 * ipus_context_destroy releases any that remain.  No reference counterpart:
 * it lets a caller check that an error path released what it allocated. */
int ipus_context_live_buffers(ipus_context *context, uint64_t *count, uint64_t *bytes);
/* Failure injection for tests of error propagation (the role of the
 * reference's device timeouts and retry path, crates/ipu-tests/src/
 * main.rs:985-1006, without a device fault): after `launches_before` more
 * ipus_launch calls on this context, the next one returns `status` (< 0)
 * without enqueuing work and the injection clears; status 0 cancels. */
int ipus_context_inject_launch_failure(ipus_context *context, uint32_t launches_before,
                                       int status);
/* Stream-ordered device copy and byte fill. */
int ipus_buffer_copy(ipus_context *context, void *device_dst, const void *device_src,
                     size_t bytes);
int ipus_buffer_memset(ipus_context *context, void *device_pointer, int value, size_t bytes);

/* ---- synchronisation and timing ---- */
int ipus_stream_sync(ipus_context *context);
typedef struct ipus_event ipus_event;
int ipus_event_create(ipus_context *context, ipus_event **event);
int ipus_event_destroy(ipus_event *event);
int ipus_event_record(ipus_context *context, ipus_event *event);
int ipus_event_elapsed_ms(ipus_event *start, ipus_event *end, float *milliseconds);

/* ---- kernel ABI registry (tile_kernel_abi, kernel.rs:1215-1382) ----
 *
 * Symbols (output, inputs, u32 scalars in order):
 *   ipu_stack_gemm_f16                 out f16 [B,M,N]; left, right f16;
 *        batches, rows, columns, inner, transpose_left, transpose_right,
 *        left_batch_stride, right_batch_stride  (strides in elements, 0 =
 *        broadcast).  Replaces gemm_f16_amp (device/gemm_f16_amp.S:186-440)
 *        with fp32 accumulation and fp16 output.
 *   ipu_stack_gemm_f16_gelu            as ipu_stack_gemm_f16, then the tanh
 *        GELU of each fp16 result element (bit-identical to
 *        ipu_stack_gemm_f16 followed by ipu_stack_gelu_tanh_approx_f16).  No
 *        reference symbol: build_package fuses a Gemm whose result feeds only
 *        one Gelu (graph.rs:315-331) into this launch.
 *   ipu_stack_gemm_f16_accumulate      out f16 [B,M,N]; left, right, addend
 *        f16; the ipu_stack_gemm_f16 scalars, then addend_batch_stride,
 *        addend_row_stride (elements; 0 broadcasts the addend over batches /
 *        rows): out = addend + A.B with the product rounded to fp16 first
 *        and the sum formed like ipu_stack_add_f16 (fp32 add, one rounding),
 *        so it is bit-identical to ipu_stack_gemm_f16 followed by that Add.
 *        The addend may be the output itself (the reference's accumulate
 *        mode, C += A.B: device/gemm_f16_amp.S:43-52, 290-363, used after
 *        the first K block by crates/ipu-codegen/src/low.rs:3483-3486), but
 *        the output must not overlap A or B.  build_package fuses a Gemm
 *        whose result only feeds an Add into this launch.
 *   ipu_stack_gemm_f16_split           out fp32 partials
 *        float[splits][batches][rows][columns]; inputs as ipu_stack_gemm_f16;
 *        scalars as ipu_stack_gemm_f16 plus splits: split z sums k in
 *        [z c, (z + 1) c), c = 64 * ceil(ceil(inner / splits) / 64), and
 *        ceil(inner / c) must equal splits.  Needs the 256 x 256 kernel's
 *        conditions (16-byte aligned operands; columns and inner, and rows
 *        when the left operand is transposed, multiples of 8), else
 *        IPUS_ERROR_UNAVAILABLE.  No reference symbol (the reference's
 *        split-K is the ParallelReduction plan, operator.rs:307-347):
 *        build_package plans it for few-tile, long-K GEMMs.
 *   ipu_stack_reduce_splits_f16        out f16; input the fp32 partials;
 *        splits, element_count (a multiple of 8), gelu (0/1): the sum over
 *        splits in order, rounded to fp16 once (GELU of that value when
 *        gelu = 1, as in ipu_stack_gemm_f16_gelu).
 *   ipu_stack_reduce_splits_accumulate_f16  out f16; partials, addend f16;
 *        splits, batches, rows, columns, addend_batch_stride,
 *        addend_row_stride: the split sum rounded to fp16, plus the addend
 *        as in ipu_stack_gemm_f16_accumulate (columns a multiple of 8).
 *   ipu_stack_gemm_f32                 as above in fp32
 *        (device/gemm_f32_64_amp.S:125-385).
 *   ipu_stack_flash_attention_online_f16  out (f32 or f16); query, key,
 *        value f16 [streams, rows, width]; matrices, query_rows, key_rows,
 *        query_dimension, value_dimension, scale_bits (0 = 1/sqrt(width)),
 *        causal, output_f16.  Shape fields follow AttentionKernelShape
 *        (kernel.rs:121-129); semantics device/flash_attention_online_f16.cpp:
 *        68-143 plus the causal limit of crates/ipu-tests/src/diagnostic.rs:741-745.
 *   ipu_stack_flash_attention_heads_f16  as above, then query_heads,
 *        key_heads, value_heads: operand stream s is head s % h of matrix
 *        s / h of an unsplit [streams / h, rows, h * width] tensor (h = 1:
 *        contiguous; streams % h == 0).  The zero-copy form of SplitHeads
 *        (operator.rs:213-279) feeding attention; build_package emits it.
 *   Decoder serving (no reference counterpart; positions, offsets, lengths and
 *   tables are int32 device arrays that the host never reads, frequencies fp32
 *   in rad per position, e.g. ipus_rotary_frequencies; f32 scalars as bits):
 *   ipu_stack_rotary_f16, ipu_stack_rotary_f32   out; input, positions [rows],
 *        frequencies [rotary_width / 2]; rows, heads, width, rotary_width,
 *        interleaved, input_row_stride, input_head_stride, output_row_stride,
 *        output_head_stride (elements), magnitude_bits (0 = 1).  Turns pair
 *        i of every head by positions[row] * frequencies[i] (reduced in 64
 *        bits), scaled by the magnitude: elements (i, rotary_width / 2 + i),
 *        interleaved = 1: (2 i, 2 i + 1); elements from rotary_width on are
 *        copied.  fp32 arithmetic, one rounding.  The output is the input
 *        (with its strides) or does not overlap it; its own heads must not
 *        overlap.  width <= 2048, rotary_width even.
 *   ipu_stack_norm_rotary_f16, ipu_stack_norm_rotary_f32   out; input,
 *        query_weight, key_weight [width] (in the input's type), positions,
 *        frequencies; rows, query_heads, key_heads, width, rotary_width,
 *        interleaved, input_row_stride, output_row_stride, epsilon_bits,
 *        magnitude_bits.  A row's heads lie side by side, queries before keys
 *        (the value heads of a fused projection may follow in the row): each
 *        becomes x * weight / sqrt(mean(x^2) + epsilon), then is turned as
 *        above, with one rounding, in place or not as there.  key_heads or
 *        query_heads may be 0 (its weight pointer is then not read, but not
 *        null either).
 *   ipu_stack_append_pages_f16   out the cache, fp16 [pages][2][key_heads]
 *        [page_rows][width] (keys, then values); new keys and values
 *        [rows][key_heads][width] (row strides in elements), frequencies,
 *        page_table [sequences][table_columns], row_offsets [sequences + 1],
 *        lengths [sequences]; sequences, rows, key_heads, width,
 *        key_row_stride, value_row_stride, rotary_width (0: no rotation),
 *        interleaved, magnitude_bits, pages, page_rows (a power of two up to
 *        65536), table_columns.  Rows row_offsets[s] .. row_offsets[s + 1] - 1
 *        are the last of sequence s, whose length with them is lengths[s]: the
 *        i-th of n goes to position p = lengths[s] - n + i, row p % page_rows
 *        of page page_table[s][p / page_rows], its key turned by p.  Rows past
 *        row_offsets[sequences], negative positions, positions past the table
 *        and entries outside [0, pages) write nothing.  The offsets do not
 *        decrease (nor for the attention below); a page that new rows go to
 *        belongs to one sequence and stands once in its table.
 *   ipu_stack_attention_pages_f16   out f16 [rows][query_heads][width], apart
 *        from the inputs; query
 *        f16 (heads side by side, query_row_stride elements from row to row),
 *        the cache, page_table, row_offsets, lengths; sequences, rows,
 *        max_rows, query_heads, key_heads (a divisor: query head h reads key
 *        head h / (query_heads / key_heads)), width, query_row_stride, pages,
 *        page_rows, table_columns, causal, scale_bits (0 = 1 / sqrt(width);
 *        scales by which scores of finite values pass fp32 are refused).
 *        Row i of the n of sequence s reads the keys below lengths[s], when
 *        causal those up to its position lengths[s] - n + i.  Keys without a
 *        page carry no weight; a row whose weights are all zero (no key, or
 *        only scores of -inf) gives zeros; rows outside every sequence are
 *        left as they were.  Keys and values that a row may not read, past its
 *        position or the sequence's length, may hold anything; non-finite
 *        values that it reads make its output non-finite in their columns.
 *        max_rows, the most rows of a sequence (0 = rows), only picks the
 *        kernel.  fp32 scores, maxima and sums.  width <= 1024; widths
 *        that are multiples of 8 up to 256 with 16-byte aligned pointers and
 *        strides run on the matrix units.  There the second product takes
 *        probabilities to 22 bits where max_rows x the query heads of a key
 *        head are at most 16 (at 97 to 128 columns and tables of more than
 *        2560 positions 32); it may take them rounded to fp16 where they are
 *        more, and over shared keys that are read once.  Other widths and
 *        alignments: fp32.
 *   ipu_stack_attention_shared_pages_f16   the same with shared_rows behind
 *        the scalars: positions below it lie in the pages of the first
 *        sequence's table for every sequence (a shared prompt).  They are read
 *        once for all where that pays, by launches that are not recorded into
 *        a caller's graph and with max_rows x the query heads of a key head up
 *        to 32; else by each sequence.
 *   A step with drafted tokens (no reference counterpart; the batch as above).
 *   A tree's mask is u32 [rows][mask_words]: bit j % 32 of word j / 32 says that
 *   the row reads the j-th row of its sequence (its ancestors and itself); bits
 *   past the sequence's rows or the words are not read.
 *   ipu_stack_page_tables   out an int32 state: free, missing, free pages
 *        [pages] (-1 from `free` on), held [sequences], page_table [sequences]
 *        [table_columns] (-1 from held[s] on); the previous state, with
 *        previous_sequences rows, source [sequences], lengths [sequences];
 *        sequences, previous_sequences, pages, page_rows, table_columns.
 *        Sequence s goes on with row source[s] of the previous table (the first
 *        that names it; one that names none of it begins) and has pages for
 *        lengths[s] positions, at most table_columns.  Pages past that and those
 *        of rows that nobody goes on with go behind the free ones, in the order
 *        of the previous rows; what sequences need is taken from the end, the
 *        sequences in order.  missing: how many there were too few; the sequences
 *        then hold fewer (their table ends earlier).  A first state: all pages
 *        free, previous_sequences 0.  Up to 4096 sequences; the new state lies
 *        apart from the inputs.  A page is held once: no prefix is shared.
 *   ipu_stack_slot_maps   out int32 row_offsets [sequences + 1], positions [rows],
 *        slots [rows], one after the other; counts [sequences] (new rows, below 0
 *        as 0), lengths [sequences] (with them), page_table, the tree's mask;
 *        sequences, rows, pages, page_rows, table_columns, mask_words (0: none,
 *        and not read).  Offsets are cut off at `rows`.  Row i of the n of
 *        sequence s, as the offsets say, is stored at place lengths[s] - n + i: its
 *        slot is page * page_rows + row in the page, -1 where the place has no
 *        page.  Its position is the place, in a tree lengths[s] - n + how many
 *        other rows it reads (its depth), -1 below 0.  Rows behind the last
 *        sequence: position 0, slot -1.  n is what the append and the attention
 *        take from the offsets, so where the counts pass `rows`, lengths are to be
 *        those with the rows that are left (lengths[s] less the rows cut off, as
 *        many of the last ones): else the rows left stand at the last ones' places,
 *        behind keys that nobody has written.  pages x page_rows <= 2^31; the
 *        output lies apart from the inputs.
 *   ipu_stack_attention_tree_pages_f16   as ipu_stack_attention_pages_f16 with the
 *        tree's mask behind the inputs and mask_words (at least 1) in the place of
 *        causal: row i of sequence s reads the keys before its sequence's rows,
 *        below lengths[s] - n, and those of the rows that its mask names (row j's
 *        stands at lengths[s] - n + j).  A row that reads no key gives zeros.
 *        Recorded launches do not split their keys, as there.
 *   ipu_stack_adjust_logits_f16, ipu_stack_adjust_logits_f32   out [rows] of
 *        columns logits; logits, row_offsets, tokens [rows], the tree's mask,
 *        history [sequences][history_columns], history_counts [sequences][2] (the
 *        prompt's tokens, all), penalties fp32 [sequences][3] (repetition r,
 *        frequency f, presence p), bias_offsets [sequences + 1], biases
 *        [bias_entries][2] (token, fp32 bits), allowed u32 [rows][allowed_words]
 *        (bit t % 32 of word t / 32: token t); sequences, rows, columns,
 *        input_row_stride, output_row_stride (elements, at least columns),
 *        mask_words, history_columns (with rows below 2^29), bias_entries,
 *        allowed_words.  A scalar of 0
 *        says that there is no such list, which is then not read; without a mask
 *        a row's path is its sequence's rows up to itself, else those that its
 *        mask names.  With g how often a token stands in the path and the history
 *        behind the prompt: a token of prompt, history or path has its logit x
 *        divided by r (x > 0) or multiplied by it, and if g > 0 lessened by f g +
 *        p; then its bias is added (of several entries the last), so that no penalty
 *        scales it (one that is to be scaled is added in a launch before, with
 *        penalties 1, 0, 0); a token that is not allowed gets -inf, whatever it
 *        was.  fp32 arithmetic, one rounding.
 *        Tokens outside [0, columns) count for nothing (-1: a prompt's rows, whose
 *        tokens stand in the history).  Rows outside every sequence are left as
 *        they were.  The output is the input (with its stride), or its rows share
 *        no memory with the input's; nor do they with a list that is read.  Other
 *        addresses are refused.
 *   ipu_stack_keep_pages_f16   out the caches of all layers, fp16 [layers][pages][2]
 *        [key_heads][page_rows][width]; page_table, row_offsets, lengths, path
 *        [sequences][path_columns], path_counts [sequences]; sequences, rows, layers
 *        (up to 65535), key_heads, width, pages, page_rows, table_columns,
 *        path_columns.  Row path[s][i] of the new rows of sequence s moves to row i,
 *        keys and values, for i < path_counts[s]: after it the accepted drafts stand
 *        behind one another, from place lengths[s] - n on.  The path increases; it
 *        ends at an entry that does not, or is no row of the sequence.  A place
 *        without a page is neither read nor written.
 *   ipu_stack_gelu_tanh_approx_f16     out f16; input f16; element_count
 *        (kernel.rs:1251-1263; count must be even, kernel.rs:1400-1413).
 *   ipu_stack_reduce_sum_f16           out f16; initial, packed remotes f16;
 *        num_partials (= remote partial count), element_count
 *        (kernel.rs:1264-1274; partials >= 2 and count % 8 == 0,
 *        kernel.rs:1414-1423; semantics device/reduce_add_f16.S:54-70).
 *   ipu_stack_rearrange_row_major_f16  out f16; source f16 row-major;
 *        logical_rows, physical_rows, target_order (0 AmpLeft,
 *        1 AmpTransposedRight, 2 BlockMajor), logical_columns,
 *        physical_columns, row_block, column_block, matrices
 *        (kernel.rs:1340-1364; device/rearrange_f16.cpp:36-155).
 *   ipu_stack_unpack_amp_f16           out f16 row-major; source f16;
 *        matrices, logical_rows, physical_rows, logical_columns,
 *        physical_columns, source_order (0 AmpOutput, 1 AmpTransposedLeft)
 *        (kernel.rs:1319-1339; device/unpack_amp_f16.cpp:30-83).
 *   ipu_stack_transpose_f16            out f16 [B,N,M]; source f16 [B,M,N];
 *        matrices, rows, columns.  No reference symbol: the graph-level
 *        transpose of a row-major matrix (BlockMajorOrder::TransposedMatrix
 *        semantics, crates/ipu-codegen/src/storage.rs:390-401).
 *   ipu_stack_reduce_rows_f16          out f32 [rows]; source f16 logical
 *        [rows, columns]; rows, columns, source_order (3 row-major,
 *        2 block-major), row_block, column_block.  ReductionSum over the
 *        columns with fp32 accumulation (operator.rs:307-347).
 *   ipu_stack_fill_zero                out; no inputs; byte_count.  The
 *        plan's own FillZero step (arena values, fp32 partials); no reference
 *        symbol.
 *   ipu_stack_fill_zero_u64            out; no inputs; words_per_worker,
 *        remainder_workers: the reference's FillZero step as
 *        materialize_kernel_run emits it (FILL_ZERO_U64_SYMBOL,
 *        crates/ipu-target/src/emit.rs:38; scalars kernel.rs:1223-1229,
 *        1175-1176): zeroes 8 * (6 * words_per_worker + remainder_workers)
 *        bytes; remainder_workers must be < 6.
 *
 * Reference per-shape symbols.  The reference links one specialization per
 * operand shape and names it by that shape (KernelBuildPlan::from_program,
 * kernel.rs:321-328, 374-379, 506-515).  ipus_kernel_abi, ipus_launch and
 * ipus_validate_kernel_run accept those names; the suffix fixes the shape of
 * one launch of the generic kernel:
 *   ipu_stack_rearrange_row_major_to_amp_f16_o{T}_r{LR}_p{PR}_c{LC}_p{PC}
 *        out; source row-major; the reference's scalars logical_rows,
 *        physical_rows, target_order (= T), logical_columns,
 *        physical_columns (kernel.rs:1351-1361), one matrix.  The scalars'
 *        physical extents must equal the suffix, and the logical ones too
 *        unless the suffix holds 0 there (rearrangement_specialization,
 *        kernel.rs:1122-1146).  T = 2 is block-major {64, 16}, the one block
 *        shape the reference plans for this conversion (layout.rs:356-361).
 *        Replaces rearrange_amp_left_f16.S, rearrange_block_major_f16.S,
 *        rearrange_transposed_right_f16.S and rearrange_f16.cpp.
 *   ipu_stack_unpack_amp_to_row_major_f16_o{S}_r{LR}_p{PR}_c{LC}_p{PC}
 *        out row-major; source AMP-Output (S = 0) or AMP-TransposedLeft
 *        (S = 1); scalars matrices, logical_rows, physical_rows,
 *        logical_columns, physical_columns (kernel.rs:1327-1336), extents
 *        equal to the suffix (device/unpack_amp_f16.cpp:6-40).
 *   ipu_stack_flash_attention_online_f16_m{B}_q{Q}_k{K}_d{D}_v{V}_{scale:08x}
 *        out f32; query, key, value f16 row-major; no scalars
 *        (AttentionKernelShape, kernel.rs:121-129, 986-1040): non-causal,
 *        scale = the f32 with those bits.
 * Reference symbols that are not forwarded return IPUS_ERROR_TRANSLATED
 * (the tile GEMM codelets ipu_stack_gemm_{f16,f32}_{init,accumulate}_...,
 * kernel.rs:185-193, and the staged-attention codelets
 * ipu_stack_attention_{softmax,merge}_..., kernel.rs:546-640) or
 * IPUS_ERROR_UNAVAILABLE (symbols the reference itself marks Required:
 * fp8 GEMM and casts, ipu_stack_unsupported_*).
 *
 *   ipu_stack_cast_f32_f16, ipu_stack_cast_f16_f32   out; input;
 *        element_count (Cast, kernel.rs:1313-1318).
 *   ipu_stack_add_f16, ipu_stack_add_f32   out; left, right; element_count,
 *        left_broadcast_stride, right_broadcast_stride  (Add,
 *        kernel.rs:1275-1287): out[i] = left[i % L] + right[i % R] where
 *        L, R are the operand element counts given by the two strides
 *        (trailing-axis numpy broadcasting; the graph executor handles the
 *        general case).
 *
 * Roofline calibration (no counterpart in the reference; used by the bench
 * to report the clock the MFMA pipes sustain for a given operand pattern):
 *   ipus_calibrate_mfma_f16            out: u64 shader-clock cycles, u64
 *        100 MHz ticks, then blocks*256 floats; input: operand_count
 *        fragments of 8 fp16; operand_count, iterations, blocks.  Each
 *        wave issues 8*iterations v_mfma_f32_32x32x16_f16 on its fragments.
 *   ipus_calibrate_mfma_f16_16x16x32   the same with v_mfma_f32_16x16x32_f16
 *        (the form the GEMM and attention kernels issue), eight fragment
 *        pairs per lane so that consecutive MFMAs see different operands.
 *   ipus_calibrate_copy                out; input; byte_count (a multiple of
 *        16, both pointers 16-byte aligned): a plain copy with ordinary
 *        16-byte loads and stores, whose HBM traffic counters scale those of
 *        other kernels to bytes.
 */
#define IPUS_MAX_SCALARS 32

typedef struct ipus_kernel_abi_info {
  const char *symbol;
  int input_count;
  int scalar_count;
  const char *scalar_names[IPUS_MAX_SCALARS];
  int implemented; /* KernelAvailability::Implemented */
} ipus_kernel_abi_info;

int ipus_kernel_count(int *count);
int ipus_kernel_abi_at(int index, ipus_kernel_abi_info *info);
int ipus_kernel_abi(const char *symbol, ipus_kernel_abi_info *info);

/* validate_kernel_run (kernel.rs:1384-1435) without a device: the symbol
 * resolves (including the reference per-shape names above), pointer arity
 * and scalar count match its ABI, and the scalars meet its constraints
 * (even GELU count, reduce partials and count, FillZero remainder, per-shape
 * suffix agreement).  Returns 0 or the status ipus_launch would return for
 * the same call before touching the device. */
int ipus_validate_kernel_run(const char *symbol, int input_count, const uint32_t *scalars,
                             int scalar_count);

/* One ComputeStep{symbol, output_address, input_addresses, arguments}:
 * validates pointer arity and scalar constraints (validate_kernel_run,
 * kernel.rs:1384-1435) and enqueues on the context stream. */
int ipus_launch(ipus_context *context, const char *symbol, void *output,
                const void *const *inputs, int input_count, const uint32_t *scalars,
                int scalar_count);

/* ---- split-K fp16 GEMM that allocates nothing ----
 * No counterpart in the reference.  For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc): the same computation as launching
 * ipu_stack_gemm_f16_split into a caller-allocated partials buffer and then
 * ipu_stack_reduce_splits_f16 (gelu 0/1) into `output`, with the partials in
 * a device array the library holds for each device from its first context
 * until the process ends.  Arguments are those two symbols' scalars; the
 * operands and output follow ipu_stack_gemm_f16.  The partials,
 * batches * rows * columns * splits fp32 values, must fit
 * IPUS_SPLIT_SCRATCH_BYTES (16 MiB: build_package's split plans, at most 64
 * split tiles of 256 x 256, all fit), else IPUS_ERROR_UNSUPPORTED_COUNT.
 * The call enqueues on the context's stream and calls no allocator.  Every
 * call on one device shares that device's array: calls that overlap on one
 * device (from other contexts, or recorded and replayed on other streams) race;
 * those of one context stand one after the other on its stream. */
#define IPUS_SPLIT_SCRATCH_BYTES (16ull << 20)
int ipus_gemm_f16_split_noalloc(ipus_context *context, void *output, const void *left,
                                const void *right, uint32_t batches, uint32_t rows,
                                uint32_t columns, uint32_t inner, int transpose_left,
                                int transpose_right, uint64_t left_batch_stride,
                                uint64_t right_batch_stride, uint32_t splits, int gelu);

/* ---- rotary frequencies (host) ----
 * frequencies[i] = base^(-2 i / rotary_width), i < rotary_width / 2, in rad per
 * position, and the magnitude of the rotated elements, for
 * ipu_stack_rotary_* and the kernels that rotate on the way.  scaling, for
 * contexts `factor` times the trained one:
 *   PLAIN   as they are (factor is not read);
 *   LINEAR  all divided by factor (positions interpolated);
 *   BASE    of base * factor^(rotary_width / (rotary_width - 2)), which divides
 *           the slowest by factor and leaves the fastest (rotary_width > 2);
 *   BANDED  by the turns each makes over the trained_rows of training: up to
 *           slow_turns divided by factor, from fast_turns on as they are, a
 *           linear ramp between; magnitude 0.1 ln(factor) + 1 for factor > 1.
 * The magnitude is 1 otherwise.  Computed in 64 bits, rounded once. */
#define IPUS_ROTARY_PLAIN 0
#define IPUS_ROTARY_LINEAR 1
#define IPUS_ROTARY_BASE 2
#define IPUS_ROTARY_BANDED 3
int ipus_rotary_frequencies(float *frequencies, float *magnitude, uint32_t rotary_width,
                            double base, int scaling, double factor, double trained_rows,
                            double slow_turns, double fast_turns);

/* ---- synthetic inputs (host, deterministic, multithreaded) ----
 * value(seed, tensor, i) from SplitMix64(seed ^ (tensor << 48) ^ i):
 * distribution 0 = uniform [-1, 1) from the top 24 bits, 1 = normal (Box-Muller
 * on two draws), times `scale`; fp16 outputs are rounded to nearest even. */
int ipus_synth_f16(uint16_t *out, uint64_t count, uint64_t seed, uint32_t tensor,
                   int distribution, float scale);
int ipus_synth_f32(float *out, uint64_t count, uint64_t seed, uint32_t tensor,
                   int distribution, float scale);

#ifdef __cplusplus
}
#endif
#endif /* IPUS_H */
