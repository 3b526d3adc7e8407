/**
    extern(C) binding of libdopthip.so, the MI355X kernel library and host mirror behind the dopt.hip backend.
    
    GENERATED by hip/gen_shim.py from include/dopt_hip.h and include/dopt_hip_plan.h: one declaration per C
    declaration, in header order.  What each function does, and which call site of the reference's CUDA backend
    it replaces, is documented in those headers.  Written where no D compiler exists: never compiled.
*/
module dopt.hip.shim;

extern(C) @nogc nothrow:

// ---- include/dopt_hip.h
alias dopt_hip_status = int;
enum
{
    DOPT_HIP_OK = 0,
    DOPT_HIP_ERR_INVALID = 1,
    DOPT_HIP_ERR_RUNTIME = 2,
    DOPT_HIP_ERR_UNSUPPORTED = 3,
    DOPT_HIP_ERR_OOM = 4,
    DOPT_HIP_ERR_RTC = 5,
}

alias dopt_hip_dtype = int;
enum
{
    DOPT_HIP_F32 = 0,
    DOPT_HIP_I32 = 1,
}

alias dopt_hip_tiny_limits = int;
enum
{
    DOPT_HIP_TINY_SLOTS = 48,
    DOPT_HIP_TINY_NODES = 40,
    DOPT_HIP_TINY_ELEMS = 4096,
}

alias dopt_hip_tiny_kind = int;
enum
{
    DOPT_HIP_TINY_POINTWISE = 0,
    DOPT_HIP_TINY_REDUCE = 1,
    DOPT_HIP_TINY_SOFTMAX = 2,
    DOPT_HIP_TINY_SOFTMAX_GRAD = 3,
    DOPT_HIP_TINY_REPEAT = 4,
    DOPT_HIP_TINY_MATVEC = 5,
}

alias dopt_hip_activation = int;
enum
{
    DOPT_HIP_ACT_NONE = 0,
    DOPT_HIP_ACT_RELU = 1,
    DOPT_HIP_ACT_GELU = 2,
    DOPT_HIP_ACT_SILU = 3,
}

alias dopt_hip_row_norm = int;
enum
{
    DOPT_HIP_NORM_NONE = 0,
    DOPT_HIP_NORM_LAYER = 1,
    DOPT_HIP_NORM_RMS = 2,
}

struct dopt_hip_tiny_node
{
    int kind;
    int op;
    int dst;
    int a;
    int b;
    int a_kind;
    int b_kind;
    int n;
    int dst_offset;
    int a_offset;
    int b_offset;
    int[4] dims;
    int[4] reps;
}

struct dopt_hip_conv_desc
{
    size_t N;
    size_t C;
    size_t H;
    size_t W;
    size_t K;
    size_t R;
    size_t S;
    size_t padH;
    size_t padW;
    size_t strideH;
    size_t strideW;
}

struct dopt_hip_split_sum
{
    const(float)* partial;
    int splits;
    size_t elems;
    size_t C;
    size_t inner;
    const(float)* bias;
    float* value;
    int lanes;
}

struct dopt_hip_residual_norm_desc
{
    size_t rows;
    size_t cols;
    size_t gates;
    int post;
    int pre;
    float eps;
    float residual_scale;
}

struct dopt_hip_tensor_ref
{
    float* w;
    const(float)* g;
    float* m;
    float* v;
    float* vhat;
    size_t n;
    int skip_w;
}

struct dopt_hip_matrix_ref
{
    float* w;
    const(float)* g;
    float* m;
    size_t rows;
    size_t cols;
}

struct dopt_hip_gradient_ref
{
    const(float)* g;
    float* out_;
    size_t n;
}

int dopt_hip_init(int device);
int dopt_hip_shutdown();
const(char)* dopt_hip_last_error();
int dopt_hip_malloc(void** ptr, size_t bytes);
int dopt_hip_free(void* ptr);
int dopt_hip_pool_trim();
int dopt_hip_pool_stats(size_t* live_bytes, size_t* cached_bytes, size_t* device_allocs);
int dopt_hip_memset(void* dst, int byte_value, size_t bytes);
int dopt_hip_copy_h2d(void* dst, const(void)* host_src, size_t bytes);
int dopt_hip_copy_d2h(void* host_dst, const(void)* src, size_t bytes);
int dopt_hip_copy_d2d(void* dst, const(void)* src, size_t bytes);
int dopt_hip_host_alloc(void** host_ptr, size_t bytes);
int dopt_hip_host_free(void* host_ptr);
int dopt_hip_copy_h2d_async(void* dst, const(void)* pinned_src, size_t bytes);
int dopt_hip_copy_h2d_beside(void* dst, const(void)* pinned_src, size_t bytes);
int dopt_hip_upload_join();
int dopt_hip_copy_d2d_batch(int n, const(void*)* dst, const(const(void)*)* src, const(size_t)* bytes);
int dopt_hip_sync();
void* dopt_hip_stream();
int dopt_hip_event_create(void** event);
int dopt_hip_event_record(void* event);
int dopt_hip_event_elapsed_ms(void* start, void* stop, float* ms);
int dopt_hip_event_sync(void* event);
int dopt_hip_event_destroy(void* event);
int dopt_hip_pointwise(const(char)* op, int dtype, size_t n, const(void)* a, const(void)* b_or_null, void* out_);
int dopt_hip_pointwise_chain(int dtype, size_t n, size_t inner, int nin, const(const(void)*)* in_, const(ubyte)* in_kind, int nnodes, const(const(char)*)* node_op, const(int)* node_lhs, const(int)* node_rhs, void* out_);
int dopt_hip_pointwise_chain_compile_only(int dtype, int nin, const(ubyte)* in_kind, int nnodes, const(const(char)*)* node_op, const(int)* node_lhs, const(int)* node_rhs, const(char)* arch);
int dopt_hip_pointwise_arity(const(char)* op);
int dopt_hip_pointwise_index(const(char)* op);
int dopt_hip_tiny_graph(int nslots, const(void*)* slots, int nnodes, const(dopt_hip_tiny_node)* nodes);
int dopt_hip_reduce(const(char)* op, int dtype, const(size_t)* shape, int rank, const(size_t)* axes, int naxes, const(void)* in_, void* out_);
int dopt_hip_reduce_squares(const(size_t)* shape, int rank, const(size_t)* axes, int naxes, const(float)* in_, float* out_);
int dopt_hip_argmin(int dtype, const(size_t)* shape, int rank, size_t axis, const(void)* in_, int* out_);
int dopt_hip_rtc_compile_only(const(char)* op, int dtype, const(char)* arch);
int dopt_hip_slice(int rank, const(size_t)* in_shape, const(size_t)* out_shape, const(size_t)* start, const(void)* in_, void* out_);
int dopt_hip_pad(int rank, const(size_t)* in_shape, const(size_t)* out_shape, const(size_t)* before, const(void)* in_, void* out_);
int dopt_hip_repeat(int rank, const(size_t)* in_shape, const(size_t)* reps, const(void)* in_, void* out_);
int dopt_hip_transpose2d(size_t rows, size_t cols, const(void)* in_, void* out_);
int dopt_hip_sgemm(size_t M, size_t N, size_t K, const(float)* A, const(float)* B, float* C);
int dopt_hip_sgemm_t(int transA, int transB, size_t M, size_t N, size_t K, const(float)* A, const(float)* B, float* C);
int dopt_hip_sgemm_batch(int n, const(int)* transA, const(int)* transB, const(size_t)* M, const(size_t)* N, const(size_t)* K, const(const(float)*)* A, const(const(float)*)* B, const(float*)* C);
ulong dopt_hip_sgemm_order(int transA, int transB, size_t M, size_t N, size_t K);
int dopt_hip_sgemm_rank1(int transA, int transB, size_t M, size_t N, size_t K, const(float)* A, const(float)* B, const(float)* u, const(float)* v, int relu, float* C);
int dopt_hip_sgemm_relu_grad(int transA, int transB, size_t M, size_t N, size_t K, const(float)* A, const(float)* B, const(float)* x, float* C);
int dopt_hip_conv_fwd(const(dopt_hip_conv_desc)* d, const(float)* x, const(float)* w, float* y);
int dopt_hip_conv_fwd_bias(const(dopt_hip_conv_desc)* d, const(float)* x, const(float)* w, const(float)* bias, float* y);
int dopt_hip_conv_bwd_data(const(dopt_hip_conv_desc)* d, const(float)* dy, const(float)* w, float* dx);
size_t dopt_hip_conv_packed_bytes(const(dopt_hip_conv_desc)* d, int bwd_data);
int dopt_hip_conv_packed_layout(const(dopt_hip_conv_desc)* d, int bwd_data);
int dopt_hip_conv_pack_batch(int n, const(dopt_hip_conv_desc)* descs, const(int)* bwd_data, const(const(float)*)* w, const(float*)* packed);
int dopt_hip_conv_fwd_bias_packed(const(dopt_hip_conv_desc)* d, const(float)* x, const(float)* packed, const(float)* bias, float* y);
int dopt_hip_conv_bwd_data_packed(const(dopt_hip_conv_desc)* d, const(float)* dy, const(float)* packed, float* dx);
int dopt_hip_conv_fwd_bias_packed_open(const(dopt_hip_conv_desc)* d, const(float)* x, const(float)* packed, const(float)* bias, float* y, dopt_hip_split_sum* open);
int dopt_hip_conv_bwd_data_packed_open(const(dopt_hip_conv_desc)* d, const(float)* dy, const(float)* packed, float* dx, dopt_hip_split_sum* open);
int dopt_hip_conv_bwd_pair_packed_open(const(dopt_hip_conv_desc)* d, const(float)* dy, const(float)* packed, const(float)* x, float* dx, float* dw, dopt_hip_split_sum* open, dopt_hip_split_sum* open_dw);
int dopt_hip_conv_pair_probe(int enable);
int dopt_hip_conv_pair_probe_read(int* launches, double* total_us, double* flops, double* bytes);
int dopt_hip_split_sum_close(const(dopt_hip_split_sum)* open);
int dopt_hip_conv_bwd_filter(const(dopt_hip_conv_desc)* d, const(float)* dy, const(float)* x, float* dw);
int dopt_hip_conv_bwd_filter_batch(int n, const(dopt_hip_conv_desc)* descs, const(const(float)*)* dy, const(const(float)*)* x, const(float*)* dw);
int dopt_hip_maxpool_fwd(size_t N, size_t C, size_t H, size_t W, size_t ph, size_t pw, const(float)* x, float* y);
int dopt_hip_maxpool_bwd(size_t N, size_t C, size_t H, size_t W, size_t ph, size_t pw, const(float)* dy, const(float)* x, float* dx);
int dopt_hip_softmax_fwd(size_t N, size_t C, size_t inner, const(float)* x, float* y);
int dopt_hip_softmax_bwd(size_t N, size_t C, size_t inner, const(float)* dy, const(float)* y, float* dx);
int dopt_hip_relu_fwd(size_t n, const(float)* x, float* y);
int dopt_hip_relu_bwd(size_t n, const(float)* dy, const(float)* x, float* dx);
int dopt_hip_bias_fwd(size_t N, size_t C, size_t inner, const(float)* x, const(float)* b, float* y);
int dopt_hip_bias_bwd(size_t N, size_t C, size_t inner, const(float)* dy, float* db);
int dopt_hip_bias_bwd_noalloc(size_t N, size_t C, size_t inner, const(float)* dy, float* db);
int dopt_hip_uniform(ulong seed, ulong call, size_t n, float* out_);
int dopt_hip_philox_raw(ulong seed, ulong call, size_t n, uint* out_);
int dopt_hip_image_transform(size_t N, size_t C, size_t H, size_t W, size_t jitterX, size_t jitterY, const(int)* geom, const(float)* in_, float* out_);
int dopt_hip_bn_train(size_t N, size_t C, size_t inner, double momentum, const(float)* x, const(float)* scale, const(float)* bias, const(float)* run_mean, const(float)* run_var, float* packed);
int dopt_hip_bn_grad(size_t N, size_t C, size_t inner, const(float)* dy, const(float)* x, const(float)* scale, float* packed);
int dopt_hip_bn_train_relu(size_t N, size_t C, size_t inner, double momentum, const(float)* x, const(float)* scale, const(float)* bias, const(float)* run_mean, const(float)* run_var, float* packed);
int dopt_hip_bn_grad_relu(size_t N, size_t C, size_t inner, const(float)* dy, const(float)* y, const(float)* x, const(float)* scale, float* packed);
int dopt_hip_bn_grad_fused(size_t N, size_t C, size_t inner, const(float)* dy, const(float)* y, const(float)* x, const(float)* scale, float* packed, float* dx_sum);
int dopt_hip_bn_train_open(size_t N, size_t C, size_t inner, double momentum, const(dopt_hip_split_sum)* x_open, const(float)* scale, const(float)* bias, const(float)* run_mean, const(float)* run_var, float* packed, int relu);
int dopt_hip_bn_grad_open(size_t N, size_t C, size_t inner, const(dopt_hip_split_sum)* dy_open, int keep_dy, const(float)* y, const(float)* x, const(float)* scale, float* packed, float* dx_sum);
int dopt_hip_bn_train_pool(size_t N, size_t C, size_t H, size_t W, double momentum, const(float)* x, const(dopt_hip_split_sum)* x_open, const(float)* scale, const(float)* bias, const(float)* run_mean, const(float)* run_var, float* packed, int relu, float* pooled);
int dopt_hip_bn_grad_pool(size_t N, size_t C, size_t H, size_t W, const(float)* dpooled, const(float)* y, const(float)* x, const(float)* scale, float* packed, float* dx_sum);
int dopt_hip_bn_grad_side(size_t N, size_t C, size_t H, size_t W, const(float)* dy, const(dopt_hip_split_sum)* dy_open, int keep_dy, const(float)* dpooled, const(dopt_hip_split_sum)* dpooled_open, const(float)* y, const(float)* x, const(float)* scale, float* packed, float* dx_sum, const(dopt_hip_split_sum)* side);
int dopt_hip_bn_wait_limit(uint polls);
int dopt_hip_bn_infer(size_t N, size_t C, size_t inner, const(float)* x, const(float)* scale, const(float)* bias, const(float)* mean, const(float)* var, float* y);
int dopt_hip_group_norm(size_t N, size_t C, size_t inner, size_t groups, int channels_last, float eps, int act, const(float)* x, const(float)* scale, const(float)* bias, float* packed);
int dopt_hip_group_norm_grad(size_t N, size_t C, size_t inner, size_t groups, int channels_last, int act, const(float)* dy, const(float)* x, const(float)* scale, const(float)* bias, const(float)* stats, float* packed);
int dopt_hip_residual_norm(const(dopt_hip_residual_norm_desc)* desc, const(float)* x, const(float)* branch, const(float)* gate, const(float)* post_scale, const(float)* post_bias, const(float)* pre_scale, const(float)* pre_bias, float* y, float* h, float* stats);
int dopt_hip_residual_norm_grad(const(dopt_hip_residual_norm_desc)* desc, const(float)* dy, const(float)* dh, const(float)* y, const(float)* branch, const(float)* gate, const(float)* post_scale, const(float)* post_bias, const(float)* pre_scale, const(float)* stats, float* dx, float* dbranch, float* dgate, float* dpost_scale, float* dpost_bias, float* dpre_scale, float* dpre_bias);
int dopt_hip_dense_act(size_t M, size_t N, size_t K, int act, const(float)* x, const(float)* w, const(float)* bias, const(float)* residual, float* y, float* pre);
int dopt_hip_dense_act_grad(size_t M, size_t N, size_t K, int act, const(float)* dy, const(float)* pre, const(float)* x, const(float)* w, float* dx, float* dw, float* dbias);
int dopt_hip_dense_groups(size_t G, size_t M, size_t N, size_t K, int act, const(int)* offsets, const(float)* x, const(float)* w, const(float)* bias, float* y, float* pre);
int dopt_hip_dense_groups_grad(size_t G, size_t M, size_t N, size_t K, int act, const(int)* offsets, const(float)* dy, const(float)* pre, const(float)* x, const(float)* w, float* dx, float* dw, float* dbias);
int dopt_hip_optim_create(int ntensors, const(dopt_hip_tensor_ref)* refs, void** handle);
int dopt_hip_optim_destroy(void* handle);
int dopt_hip_sgd_step(void* handle, float lr, float mu, int nesterov);
int dopt_hip_adam_step(void* handle, float alpha, float beta1, float beta2, float eps, float* b1, float* b2);
int dopt_hip_amsgrad_step(void* handle, float alpha, float beta1, float beta2, float eps, float* b1, float* b2);
int dopt_hip_sgd_step_scaled(void* handle, float lr, float mu, int nesterov, const(float)* factor);
int dopt_hip_adam_step_scaled(void* handle, float alpha, float beta1, float beta2, float eps, float* b1, float* b2, const(float)* factor);
int dopt_hip_amsgrad_step_scaled(void* handle, float alpha, float beta1, float beta2, float eps, float* b1, float* b2, const(float)* factor);
int dopt_hip_muon_create(int nmatrices, const(dopt_hip_matrix_ref)* refs, void** handle);
int dopt_hip_muon_destroy(void* handle);
int dopt_hip_muon_step(void* handle, float lr, float mu, int nesterov, float decay, int iterations);
int dopt_hip_muon_step_scaled(void* handle, float lr, float mu, int nesterov, float decay, int iterations, const(float)* factor);
int dopt_hip_gradient_norm_create(int ntensors, const(dopt_hip_gradient_ref)* refs, void** handle);
int dopt_hip_gradient_norm_destroy(void* handle);
int dopt_hip_gradient_norm(void* handle, float max_norm, float* result);
int dopt_hip_gradient_clip(void* handle, float max_norm, float* result);

// ---- include/dopt_hip_plan.h
enum
{
    DOPT_HIP_PLAN_VIEWS = 1,
    DOPT_HIP_PLAN_TIMING = 2,
    DOPT_HIP_PLAN_TIMING_SHAPES = 64,
    DOPT_HIP_PLAN_FUSE = 4,
    DOPT_HIP_PLAN_GRAPH = 16,
    DOPT_HIP_PLAN_OVERLAP = 8,
    DOPT_HIP_PLAN_OVERLAP_LIGHT = 32,
}

struct dopt_hip_kernel
{
    void* self;
    int function(void* self, int ninputs, const(const(void)*)* inputs, const(size_t)* input_bytes, void* output, size_t output_bytes) execute;
    void function(void* self) destroy;
}

alias dopt_hip_kernel_ctor = int function(void* graph, int op, void* user, dopt_hip_kernel* out_);
int dopt_hip_graph_create(void** graph);
int dopt_hip_graph_destroy(void* graph);
int dopt_hip_graph_add_op(void* graph, const(char)* op_type, int dtype, int rank, const(size_t)* shape, int ndeps, const(int)* deps, int* op_id);
int dopt_hip_graph_set_attr_sizes(void* graph, int op, const(char)* key, const(size_t)* values, int n);
int dopt_hip_graph_set_attr_double(void* graph, int op, const(char)* key, double value);
int dopt_hip_graph_value(void* graph, int op, void** device_ptr, size_t* bytes);
int dopt_hip_graph_op_type(void* graph, int op, const(char)** op_type, int* dtype, int* rank, size_t* shape8, int* ndeps);
int dopt_hip_graph_op_dep(void* graph, int op, int index, int* dep);
int dopt_hip_register_kernel(const(char)* op_name, dopt_hip_kernel_ctor ctor, void* user);
int dopt_hip_deregister_kernel(const(char)* op_name);
int dopt_hip_list_operations(char* buf, size_t buf_bytes, size_t* needed);
int dopt_hip_plan_create(void* graph, int noutputs, const(int)* outputs, uint flags, void** plan);
int dopt_hip_plan_execute(void* plan, int nargs, const(int)* arg_ops, const(const(void)*)* arg_ptrs, const(int)* arg_on_host, int nrets, const(void*)* rets);
int dopt_hip_plan_result(void* plan, int op, void** device_ptr, size_t* bytes);
int dopt_hip_plan_stats(void* plan, size_t* kernels, size_t* buffer_bytes);
int dopt_hip_plan_recordings(void* plan, size_t* recorded, size_t* replays);
int dopt_hip_plan_profile(void* plan, char* buf, size_t buf_bytes, size_t* needed);
int dopt_hip_plan_destroy(void* plan);
